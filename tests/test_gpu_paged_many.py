"""Attention of many query rows a kv head over long contexts of a paged cache (bf16, head_d <= 128): tiles
of 64, 128 and 256 rows, items whole and in ranges, prefixes beside them, against the definition in
float64; and both sides of what decides whether a prefix is read once."""
import numpy as np
import pytest

import cache_helpers as C
import paged_helpers as P

pytestmark = pytest.mark.gpu


def run(am, p, **kw):
    am.paged_attention_ex(p.cache, p.drafts, p.out.dev, p.lse, prefix=p.prefix, **kw)


@pytest.mark.parametrize("D", [8, 16, 24, 64, 72, 80, 120, 128])
@pytest.mark.parametrize("T", [17, 33, 65, 100, 130, 257])
def test_rows_of_a_tile(am, dev, D, T):
    """From 34 rows (one tile of 64) to 514 (three of 256); lengths that end inside a block."""
    p = P.Paged(am, "bf16", 2, 4, 2, T, D, 16, [777, 401], [T, T - 9], slots=80)
    run(am, p)
    p.check()


@pytest.mark.parametrize("B,Hq,G,T", [(16, 16, 16, 40), (16, 32, 16, 60), (32, 8, 8, 129), (5, 70, 14, 40),
                                      (17, 16, 16, 64)])
def test_items_whole(am, dev, B, Hq, G, T):
    """Enough pairs of sequence and kv head that workgroups take whole items, few rows of them full."""
    rng = np.random.default_rng(B * T)
    lens = [int(x) for x in rng.integers(0, 150, B)]
    counts = [int(x) for x in rng.integers(0, T + 1, B)]
    p = P.Paged(am, "bf16", B, Hq, G, T, 64, 32, lens, counts, slots=24)
    run(am, p)
    p.check()


@pytest.mark.parametrize("lens", [[0], [1], [63], [64], [65], [127], [128], [129], [2000]])
@pytest.mark.parametrize("T", [40, 100, 200])
def test_lengths(am, dev, T, lens):
    for D in (64, 128):
        p = P.Paged(am, "bf16", 1, 2, 1, T, D, 64, lens, slots=40)
        run(am, p)
        p.check()


@pytest.mark.parametrize("page", [16, 32, 48, 80, 256])
def test_pages(am, dev, page):
    p = P.Paged(am, "bf16", 3, 4, 2, 45, 96, page, [600, 3, 129], [45, 0, 30], slots=-(-1024 // page))
    run(am, p)
    p.check()


@pytest.mark.parametrize("order,offset,pad", [("rows", 0, 0), ("heads", 8, 8), ("rows", 16, 24)])
@pytest.mark.parametrize("T", [24, 80])
def test_strides(am, dev, order, offset, pad, T):
    p = P.Paged(am, "bf16", 3, 4, 2, T, 128, 16, [60, 700, 99], first=[0, 3], rows=[50], order=order,
                offset=offset, pad=pad, slots=64)
    run(am, p)
    p.check()


@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("T,rows", [(1, 400), (3, 600), (20, 900), (70, 1500), (70, 200)])
def test_prefixes_beside_rows_of_their_own(am, dev, D, T, rows):
    """Prefixes of many query rows, their members' own rows many or few; the last group has no prefix,
    and sequence 0 is in none."""
    B = 9
    lens = [rows + 5 + 31 * b for b in range(B)]
    p = P.Paged(am, "bf16", B, 8, 2, T, D, 16, lens, [max(0, T - b % 2) for b in range(B)],
                first=[1, 5, 7, 9], rows=[rows, rows - 13, 0], slots=160)
    run(am, p)
    p.check()


def test_a_long_table_beside_few_rows(am, dev):
    """Prefixes of many query rows in a launch of their own, sequences of few rows in another."""
    B = 14
    for D, R in ((128, 8), (64, 4)):
        for slots in (4096, 64):
            p = P.Paged(am, "bf16", B, R * 2, 2, 4, D, 16, [600 + 7 * b for b in range(B)],
                        first=[0, B], rows=[590], slots=slots)
            run(am, p)
            p.check()


@pytest.mark.parametrize("dtype,es", [("bf16", 2), ("f32", 4)])
@pytest.mark.parametrize("D", [64, 384])
def test_both_sides_of_reading_a_prefix_once(am, dev, dtype, es, D):
    """A prefix whose rows, over all members, are few beside the parts that sharing makes is read as rows
    of each member; one token more and it is shared."""
    B, T, rep = 4, 10, 2
    edge = B * rep * T * 8 // ((B - 1) * es)
    for rows in (edge - 1, edge, edge + 1, edge + 2):
        p = P.Paged(am, dtype, B, 2 * rep, 2, T, D, 16, [rows + 3 * b for b in range(B)], first=[0, B],
                    rows=[rows], slots=40)
        run(am, p)
        p.check()


@pytest.mark.parametrize("fill", [np.inf, -np.inf, 3e38])
@pytest.mark.parametrize("T", [40, 90, 150])
def test_what_no_token_attends(am, dev, fill, T):
    for D in (64, 128):
        p = P.Paged(am, "bf16", 3, 4, 2, T, D, 16, [400, 710, 333], [T, T - 7, 0], first=[0, 2],
                    rows=[395], fill=fill, slots=64)
        run(am, p)
        p.check()


@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("rows", [None, [500]])
def test_not_finite_values_reach_their_rows_alone(am, dev, D, rows):
    """In the draft's values, and in those of rows that all attend."""
    T, lens = 70, [520, 611]
    p = P.Paged(am, "bf16", 2, 2, 1, T, D, 16, lens, first=None if rows is None else [0, 2], rows=rows,
                slots=64)
    run(am, p)
    p.check()
    before, lse = p.out.numpy(), p.lse.numpy()
    V = p.V.host.copy()
    put = [(0, 2, 3, np.inf), (0, 40, 3, -np.inf), (0, 65, D - 1, -np.inf), (1, 0, 5, np.nan),
           (1, 69, 0, np.inf), (0, -500, 6, -np.inf), (1, -601, 6, -np.inf)]  # sequence, token, dim
    for b, t, d, x in put:
        r = lens[b] + t
        V[p.table[b, r // 16], :, r % 16, d] = x
    p.V.base.upload(p.V._flat(V))
    run(am, p)
    got = p.out.numpy()
    hit = np.zeros(got.shape, bool)
    for b, t, d, x in put:
        hit[b, :, max(t, 0):, d] = True
    if rows:  # (row 10 or 20 is in the shared pages: both attend it)
        hit[..., 6] = True
    assert np.array_equal(got[~hit], before[~hit]) and np.array_equal(p.lse.numpy(), lse)
    assert np.isposinf(got[0, :, 2:40, 3]).all() and np.isnan(got[0, :, 40:, 3]).all()
    assert np.isneginf(got[0, :, 65:, D - 1]).all() and np.isnan(got[1, :, :, 5]).all()
    assert np.isposinf(got[1, :, 69:, 0]).all() and np.isneginf(got[..., 6]).all()


@pytest.mark.parametrize("bad", [-1, 1 << 30, -(1 << 31)])
@pytest.mark.parametrize("T", [40, 140])
def test_rows_without_a_page(am, dev, bad, T):
    """Rows of an entry that names no page are not attended; the others are."""
    D, page = 80, 16
    p = P.Paged(am, "bf16", 2, 1, 1, T, D, page, [700, 64], slots=64)
    table = p.table.copy()
    table[0, 2] = table[0, 3] = table[0, 30] = bad
    table[1, :4] = bad
    p.tab.upload(table)
    run(am, p)
    got, got_lse = p.out.numpy(), p.lse.numpy()
    for b in range(2):
        for t in (0, 17, T - 1):
            r = np.arange(p.lens[b] + t + 1)
            r = r[(table[b, r // page] >= 0) & (table[b, r // page] < p.K.host.shape[0])]
            k, v = (x.host[table[b, r // page], 0, r % page].astype(np.float64)[None, None]
                    for x in (p.K, p.V))
            want, lse, info = C.attend64(p.Q.host[b:b + 1, :, t:t + 1], k, v, None, None, [len(r)], [1])
            tol, tol_lse = C.attend_tol("bf16", D, want, info)
            assert (np.abs(got[b, :, t] - want[0, :, 0]) <= tol[0, :, 0]).all()
            assert (np.abs(got_lse[b, :, t] - lse[0, :, 0]) <=
                    tol_lse[0, :, 0] + 4 * C.U32 * np.abs(lse[0, :, 0])).all()


def test_tokens_that_attend_nothing(am, dev):
    for T in (40, 140):
        for first in (None, [0, 2]):
            p = P.Paged(am, "bf16", 2, 2, 2, T, 64, 16, [640, 640], first=first,
                        rows=None if first is None else [500], slots=64)
            p.tab.upload(np.full(p.table.shape, -1))
            run(am, p)
            assert (p.out.numpy() == 0).all() and np.isneginf(p.lse.numpy()).all()


def test_scores_that_are_not_finite(am, dev):
    T = 60
    p = P.Paged(am, "bf16", 2, 1, 1, T, 64, 16, [600, 700], seed=6, slots=64)
    q = np.abs(p.Q.host)
    p.Q.base.upload(p.Q._flat(q))
    K = p.K.host.copy()
    K[p.table[0, 0], 0, 3] = -np.inf
    r = 700 + 1
    K[p.table[1, r // 16], 0, r % 16, 0] = np.nan
    p.K.base.upload(p.K._flat(K))
    run(am, p)
    got, lse = p.out.numpy(), p.lse.numpy()
    assert np.isnan(got[1, :, 1:]).all() and np.isnan(lse[1, :, 1:]).all()
    assert np.isfinite(got[1, :, 0]).all() and np.isfinite(got[0]).all()
    rows = np.array([i for i in range(601) if i != 3])
    k, v = (x[p.table[0, rows // 16], :, rows % 16].transpose(1, 0, 2)[None].astype(np.float64)
            for x in (K, p.V.host))
    want, wl, info = C.attend64(q[:1, :, :1], k, v, None, None, [600], [1])
    tol, _ = C.attend_tol("bf16", 64, want, info)
    assert (np.abs(got[:1, :, :1] - want) <= tol).all()


@pytest.mark.parametrize("T", [40, 100, 200])
def test_large_logits(am, dev, T):
    p = P.Paged(am, "bf16", 2, 4, 2, T, 128, 16, [600, 710], first=[0, 2], rows=[560], sigma=30.0,
                slots=64)
    run(am, p)
    p.check()


@pytest.mark.parametrize("T", [8, 40])
def test_lists_of_any_content(am, dev, T):
    rng = np.random.default_rng(7)
    p = P.Paged(am, "bf16", 6, 8, 2, T, 128, 16, [650, 760, 670, 780, 690, 740], first=[0, 3, 6],
                rows=[648, 633], slots=80)
    run(am, p)
    p.check()
    first, rows = p.prefix.first, p.prefix.rows
    for f, n in (([5, 0, 9], [1 << 30, -4]), ([-3, 1 << 30, 0], [1 << 30, 1 << 30]),
                 ([0, 6, 0], [64, 1 << 20]), ([6, 6, 6], [10, 10]), ([0, 6, 6], [1 << 30, 5]),
                 ([0, 4, 2], [700, 700])):
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
    rows.upload(np.array([648, 633]))
    run(am, p)
    p.check()


def test_same_bits_every_time(am, dev):
    for T in (40, 150):
        p = P.Paged(am, "bf16", 4, 8, 2, T, 128, 16, [900, 1500, 700, 650], first=[0, 4], rows=[600])
        run(am, p)
        first, lse = p.out.base.bits(), p.lse.bits()
        for _ in range(4):
            run(am, p)
            assert np.array_equal(p.out.base.bits(), first) and np.array_equal(p.lse.bits(), lse)


@pytest.mark.parametrize("slots", [60, 800])
@pytest.mark.parametrize("prefix", [False, True])
def test_workspaces(am, dev, prefix, slots):
    """A kv head a launch where the workspace is small; whole items where it holds no parts, or where
    they are short."""
    import hip_rt
    p = P.Paged(am, "bf16", 3, 8, 4, 40, 128, 16, [700, 800, 600], first=[0, 3] if prefix else None,
                rows=[500] if prefix else None, slots=slots)
    need = am.paged_attention_workspace_bytes(p.cache, p.drafts, p.prefix)
    ws = hip_rt.DeviceArray((need + 4096,), "bf16", fill=0)
    guard = np.full(2048, 3, np.uint16)
    tail = hip_rt.DeviceArray.view(ws, need // 2, (2048,))
    tail.upload(guard)
    size, ran = need, 0
    while size > 40960:
        w = hip_rt.DeviceArray.wrap(ws.ptr, (size // 2,), "bf16", keep=ws)
        p.out.base.upload(p.out._flat(np.full(p.out.host.shape, 7.0, np.float32)))
        try:
            run(am, p, workspace=w)
        except am.AtnError as e:
            assert prefix and e.status == -8
            break
        ran += 1
        p.check()
        assert np.array_equal(tail.bits(), guard)
        size = 40960 + (size - 40960) // 2 // 16 * 16
    assert ran >= 1 or not prefix and slots == 60
    if not prefix:  # nothing but what the library keeps for every call
        run(am, p, workspace=hip_rt.DeviceArray.wrap(ws.ptr, (20480,), "bf16", keep=ws))
        p.check()


def test_captured_and_on_two_streams(am, dev):
    """Lengths, counts and prefixes that change between replays; eager calls beside them."""
    import hip_rt
    p = P.Paged(am, "bf16", 3, 8, 2, 48, 128, 16, [900, 820, 850], [48, 30, 48], first=[0, 3], rows=[700],
                slots=80)
    o = P.Paged(am, "bf16", 2, 8, 2, 48, 64, 16, [900, 1000], seed=4)
    s, s2 = hip_rt.Stream(), hip_rt.Stream()
    call = am.paged_attention_call(p.cache, p.drafts, p.out.dev, p.lse, prefix=p.prefix)
    call(s)
    s.synchronize()
    g = hip_rt.Graph(s, lambda: call(s))
    for rows in (700, 0, 64, 688):
        p.prefix.rows.upload(np.array([rows]))
        for _ in range(2):
            g.launch()
            run(am, o, stream=s2)
        s.synchronize()
        s2.synchronize()
        p.check()
        o.check()
    g.destroy()
    for x in (s, s2):
        x.destroy()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [264, 320, 1032, 4096])
@pytest.mark.parametrize("T", [40, 60, 120])
def test_tiles_of_large_heads(am, dev, dtype, D, T):
    """head_d > 256: tiles of 32 and 64 rows, with pages of whole and of odd runs, prefixes beside."""
    for page in (16, 20):
        p = P.Paged(am, dtype, 3, 1, 1, T, D, page, [500, 333, 470], [T, T - 20, T], first=[0, 2],
                    rows=[320])
        run(am, p)
        p.check()


@pytest.mark.parametrize("B,groups", [(130, 65), (70, 70)])
@pytest.mark.parametrize("D", [64, 128])
def test_many_groups_of_many_rows(am, dev, B, groups, D):
    """More groups than a wave has lanes."""
    rng = np.random.default_rng(B)
    lens = [int(x) for x in rng.integers(520, 560, B)]
    first = [i * B // groups for i in range(groups + 1)]
    rows = [int(x) for x in rng.integers(0, 521, groups)]
    for T in (2, 40):
        p = P.Paged(am, "bf16", B, 2, 1, T, D, 16, lens, first=first, rows=rows)
        run(am, p)
        p.check()


@pytest.mark.parametrize("D", [40, 80, 64, 128])
@pytest.mark.parametrize("T", [40, 120])
def test_several_items_a_workgroup(am, dev, D, T):
    """Ranges that hold an item's end and the next one's beginning, rows of few pieces."""
    rng = np.random.default_rng(D + T)
    lens = [int(x) for x in rng.integers(0, 200, 75)]
    p = P.Paged(am, "bf16", 75, 4, 4, T, D, 16, lens, slots=512)
    run(am, p)
    p.check()


def test_overlapping_groups(am, dev):
    for first in ([0, 6, 0, 6], [0, 4, 2, 6]):
        p = P.Paged(am, "bf16", 6, 4, 2, 40, 128, 16, [600 + b for b in range(6)], first=[0, 6],
                    rows=[590], slots=64)
        p.prefix = am.SharedPrefix(C.ints(first), C.ints([590] * (len(first) - 1)))
        run(am, p)
        p.check()


@pytest.mark.parametrize("D,T,Hq,G,rows", [(128, 300, 8, 2, None), (64, 40, 4, 2, None), (80, 20, 4, 1, [896]),
                                           (128, 20, 4, 2, [1504])])
def test_many_values_that_are_not_finite(am, dev, D, T, Hq, G, rows):
    """Infinities and NaN all over: in the dims of what a token attends, and nowhere else."""
    lens = [1700, 1623, 1580]
    first = None if rows is None else [0, 3]
    p = P.Paged(am, "bf16", 3, Hq, G, T, D, 32, lens, [T, T - 6, 1], first=first, rows=rows, slots=70)
    run(am, p)
    p.check()
    before, lse = p.out.numpy(), p.lse.numpy()
    rng = np.random.default_rng(D + T)
    V = p.V.host.copy()
    hit = np.zeros(before.shape, bool)
    for b in range(3):
        for _ in range(60):
            r = int(rng.integers(lens[b] - (30 if rng.random() < 0.5 else 900), lens[b] + p.counts[b]))
            g, d = int(rng.integers(0, G)), int(rng.integers(0, D))
            page = p.table[b, r // 32]
            V[page, g, r % 32, d] = rng.choice([np.inf, -np.inf, np.nan])
            for m in range(3):  # (a shared page is every member's)
                if p.table[m, r // 32] == page:
                    hit[m, g * Hq // G:(g + 1) * Hq // G, max(0, r - lens[m]):p.counts[m], d] = True
    p.V.base.upload(p.V._flat(V))
    run(am, p)
    got = p.out.numpy()
    assert np.array_equal(np.isfinite(got), ~hit)
    assert np.array_equal(got[~hit], before[~hit]) and np.array_equal(p.lse.numpy(), lse)


@pytest.mark.parametrize("T,lens,slots", [(512, [3000, 2990], 240), (40, [3000, 1], 240), (200, [60, 900], 2000)])
def test_tails_of_any_content_cost_nothing(am, dev, T, lens, slots):
    """What lies behind a sequence's rows costs no more where it holds NaN or infinities.  (Rows' values
    looked at one key after another for each row would take 20 to 100 times the call.)"""
    import time

    import hip_rt

    def least(fill):
        p = P.Paged(am, "bf16", 2, 8, 2, T, 128, 16, lens, fill=fill, slots=slots)
        call = am.paged_attention_call(p.cache, p.drafts, p.out.dev, p.lse)
        times = []
        for _ in range(7):
            hip_rt.synchronize()
            t0 = time.perf_counter()
            for _ in range(3):
                call()
            hip_rt.synchronize()
            times.append(time.perf_counter() - t0)
        return min(times)

    plain = least(0.0)
    for fill in (np.nan, -np.inf):
        assert least(fill) < 4 * plain
