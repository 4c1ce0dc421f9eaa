"""The key/value cache of a decoding program on the GPU: commit, weights, eviction, lengths, and
a run of them with the attention that reads the cache."""
import numpy as np
import pytest

import cache_helpers as C

pytestmark = pytest.mark.gpu


class Cache:
    """A cache with host copies of everything."""

    def __init__(self, am, dtype, B, G, cap, D, lens, seen=None, order="heads", offset=0, pad=0,
                 seed=1, fill=None):
        rng = np.random.default_rng(seed)
        k, v = (rng.standard_normal((B, G, cap, D)).astype(np.float32) for _ in range(2))
        if fill is not None:
            for b in range(B):
                k[b, :, lens[b]:] = fill
                v[b, :, lens[b]:] = fill
        lay = dict(order=order, offset=offset, pad=pad)
        self.dtype, self.shape, self.lens = dtype, (B, G, cap, D), list(lens)
        self.K, self.V = C.Tensor(k, dtype, **lay), C.Tensor(v, dtype, **lay)
        self.seen = [l + 3 for l in lens] if seen is None else list(seen)
        self.weight = rng.random((B, G, cap)).astype(np.float32)
        self.pos = np.argsort(rng.random((B, G, cap)), -1).astype(np.int32)
        self.d_len, self.d_seen = C.ints(lens), C.ints(self.seen)
        self.d_weight, self.d_pos = C.floats(self.weight), C.ints(self.pos)
        self.desc = am.KvCache(self.K.dev, self.V.dev, self.d_len, self.d_seen, self.d_weight,
                               self.d_pos)

    def same(self, K, V, weight, pos):
        import hip_rt
        hip_rt.synchronize()
        assert np.array_equal(self.K.numpy(), K, equal_nan=True)
        assert np.array_equal(self.V.numpy(), V, equal_nan=True)
        assert np.array_equal(self.d_weight.numpy(), weight, equal_nan=True)
        assert np.array_equal(self.d_pos.numpy(), pos)


# ---------------------------------------------------------------- commit and advance
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,order,offset,pad", [
    (1, "heads", 0, 0), (64, "heads", 0, 0), (77, "rows", 0, 0), (128, "rows", 1, 0),
    (128, "rows", 8, 8), (520, "heads", 0, 3), (1024, "rows", 0, 0), (8192, "heads", 0, 0)])
def test_commit(am, dev, dtype, D, order, offset, pad):
    print(f"[case] commit {dtype} {D} {order} {offset} {pad}", flush=True)
    B, G, cap, T, n = 4, 3, 40, 9, 5
    c = Cache(am, dtype, B, G, cap, D, [0, 17, 37, 40], order=order, offset=offset, pad=pad)
    rng = np.random.default_rng(2)
    kd, vd = (C.Tensor(rng.standard_normal((B, G, T, D)), dtype, order, offset, pad)
              for _ in range(2))
    counts, accepted = [9, 9, 6, 9], [5, 0, 4, 5]
    path = np.array([[0, 2, 3, 7, 8], [1, 2, 3, 4, 5], [1, 4, 9, 5, 2], [8, 7, 6, 5, 4]])
    d = am.Drafts(kd.dev, kd.dev, vd.dev, count=C.ints(counts))
    for p, a in ((path, accepted), (None, accepted), (None, None), (path, None),
                 (path, [1 << 30, -3, 99, 1])):
        K, V, weight, pos = c.K.numpy(), c.V.numpy(), c.d_weight.numpy(), c.d_pos.numpy()
        pl = n if p is not None else T
        rows = C.accepted_rows(None if p is None else p.tolist(), a, counts, c.lens, cap, pl)
        for b, m in enumerate(rows):
            for i in range(m):
                t = i if p is None else p[b][i]
                K[b, :, c.lens[b] + i], V[b, :, c.lens[b] + i] = kd.host[b, :, t], vd.host[b, :, t]
                weight[b, :, c.lens[b] + i] = 0
                pos[b, :, c.lens[b] + i] = c.seen[b] + i
        args = (None if p is None else C.ints(p), None if a is None else C.ints(a))
        am.cache_commit_ex(c.desc, d, *args)
        c.same(K, V, weight, pos)
        assert c.d_len.numpy().tolist() == c.lens
        am.cache_advance_ex(c.desc, d, *args)
        c.lens = [l + m for l, m in zip(c.lens, rows)]
        c.seen = [s + m for s, m in zip(c.seen, rows)]
        assert c.d_len.numpy().tolist() == c.lens and c.d_seen.numpy().tolist() == c.seen
        c.lens = [0, 17, 37, 40]
        c.d_len.upload(np.array(c.lens, np.int32))
    for bad in ([5, 9, 9, 9], [-1] * 4):  # drafts that do not exist end a path
        p = np.stack([[0, b, 1, 2, 3] for b in bad])
        rows = C.accepted_rows(p.tolist(), None, counts, c.lens, cap, n)
        am.cache_advance_ex(c.desc, d, C.ints(p))
        assert c.d_len.numpy().tolist() == [l + m for l, m in zip(c.lens, rows)]
        c.d_len.upload(np.array(c.lens, np.int32))
    am.cache_advance_ex(c.desc, limit=20)
    assert c.d_len.numpy().tolist() == [0, 17, 20, 20]


def test_commit_long_paths(am, dev):
    """Paths longer than a wave, ending at the first entry that names no draft."""
    B, G, cap, D, T = 3, 2, 300, 32, 256
    c = Cache(am, "bf16", B, G, cap, D, [3, 0, 100])
    rng = np.random.default_rng(2)
    kd, vd = (C.Tensor(rng.standard_normal((B, G, T, D)), "bf16") for _ in range(2))
    path = np.stack([rng.permutation(T) for _ in range(B)])
    path[0, 130] = 256
    path[1, 64] = -1
    d = am.Drafts(kd.dev, kd.dev, vd.dev)
    K, V, weight, pos = (x.copy() for x in (c.K.host, c.V.host, c.weight, c.pos))
    for b, m in enumerate((130, 64, 200)):
        rows = slice(c.lens[b], c.lens[b] + m)
        K[b, :, rows], V[b, :, rows] = kd.host[b][:, path[b, :m]], vd.host[b][:, path[b, :m]]
        weight[b, :, rows] = 0
        pos[b, :, rows] = c.seen[b] + np.arange(m)
    am.cache_commit_ex(c.desc, d, C.ints(path))
    am.cache_advance_ex(c.desc, d, C.ints(path))
    c.same(K, V, weight, pos)
    assert c.d_len.numpy().tolist() == [133, 64, 300]


# ---------------------------------------------------------------- weights
def weigh64(Q, K, lse, path, rows, lens, scale):
    """Weights added to every row, and what their tolerance takes: per row the sum of
    p (score error + lse error) and of p."""
    B, H, T, D = Q.shape
    G, cap = K.shape[1:3]
    add, err = np.zeros((B, G, cap)), np.zeros((B, G, cap))
    for b in range(B):
        for h in range(H):
            g = h // (H // G)
            for i in range(rows[b]):
                t = i if path is None else path[b][i]
                if np.isneginf(lse[b, h, t]):
                    continue
                n = lens[b] + i + 1
                k, q = K[b, g, :n].astype(np.float64), Q[b, h, t].astype(np.float64)
                s = k @ q * scale
                p = np.exp(s - lse[b, h, t].astype(np.float64))
                info = dict(sabs=np.abs(k) @ np.abs(q) * abs(scale),
                            smax=np.maximum(np.abs(s), abs(lse[b, h, t])))
                add[b, g, :n] += p
                err[b, g, :n] += p * (np.expm1(C.score_error(D, info)) + 16 * C.U32)
    return add, err


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,Hq,G,T,D,lens,layout", [
    (1, 1, 1, 1, 1, [0], {}), (2, 4, 2, 1, 128, [64, 0], {}), (3, 6, 2, 7, 80, [77, 5, 130], {}),
    (2, 8, 1, 5, 64, [300, 31], dict(order="rows")), (2, 4, 4, 3, 100, [33, 34], dict(offset=1)),
    (1, 32, 4, 6, 96, [257], dict(order="rows", pad=8, offset=8)), (2, 2, 1, 12, 512, [129, 15], {}),
    (1, 4, 2, 2, 1000, [50], dict(pad=3)), (1, 2, 1, 3, 8192, [40], {}), (1, 16, 2, 40, 72, [90], {}),
    (2, 71, 1, 4, 256, [48, 47], {}), (1, 3, 3, 200, 48, [20], {}),
    (65, 16, 8, 2, 264, list(range(65)), {}), (33, 36, 9, 10, 260, list(range(40, 73)), {})])
def test_weights(am, dev, dtype, B, Hq, G, T, D, lens, layout):
    import hip_rt
    print(f"[case] weigh {dtype} {(B, Hq, G, T, D)} {lens} {layout}", flush=True)
    cap = max(lens) + T + 3
    c = Cache(am, dtype, B, G, cap, D, lens, fill=np.nan, **layout)
    rng = np.random.default_rng(3)
    q, kd, vd = (C.Tensor(rng.standard_normal((B, h, T, D)), dtype, **layout) for h in (Hq, G, G))
    counts = [T - (T // 3) * (b % 2) for b in range(B)]
    n = max(1, min(T, 7)) if T < 100 else T
    path = np.stack([np.resize(rng.permutation(k), n) for k in counts])
    accepted = ([n, max(1, n - 2), n] * B)[:B]
    d = am.Drafts(q.dev, kd.dev, vd.dev, count=C.ints(counts))
    rows = C.accepted_rows(path.tolist(), accepted, counts, lens, cap, n)
    lse = (rng.standard_normal((B, Hq, T)) + np.log(max(lens) + 1)).astype(np.float32)
    lse[:, :, 0] = -np.inf  # a token that attended nothing
    args = (C.ints(path), C.ints(accepted))
    am.cache_commit_ex(c.desc, d, *args)
    K, before = c.K.numpy(), c.d_weight.numpy()
    add, err = weigh64(q.host, K, lse, path.tolist(), rows, lens, 1.0 / np.sqrt(D))
    other = C.floats(rng.random((B, G, cap)) * 4)
    for given, start in (("own", before), (other, other.numpy()), (None, np.zeros_like(before))):
        c.d_weight.upload(before)
        am.cache_weigh_ex(c.desc, d, C.floats(lse), *args, weight_in=given)
        hip_rt.synchronize()
        got = c.d_weight.numpy()
        for b in range(B):
            m = lens[b] + rows[b]
            want = start[b, :, :m] + add[b, :, :m]
            terms = Hq // G * rows[b] + 2
            tol = 1.01 * err[b, :, :m] + terms * C.U32 * want
            assert (np.abs(got[b, :, :m] - want) <= tol).all()
            assert np.array_equal(got[b, :, m:], before[b, :, m:])  # rows behind


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f32", 128), ("bf16", 640)])
def test_weights_of_attention(am, dev, dtype, D):
    """With the attention's own lse, one token's weights add up to the group's heads."""
    import hip_rt
    B, Hq, G, cap = 2, 8, 2, 700
    c = Cache(am, dtype, B, G, cap, D, [650, 99])
    rng = np.random.default_rng(3)
    q, kd, vd = (C.Tensor(rng.standard_normal((B, h, 1, D)) * 2, dtype) for h in (Hq, G, G))
    d = am.Drafts(q.dev, kd.dev, vd.dev)
    lse = C.floats(np.zeros((B, Hq, 1)))
    am.tree_attention_ex(c.desc, d, lse=lse)
    am.cache_commit_ex(c.desc, d)
    am.cache_weigh_ex(c.desc, d, lse, weight_in=None)
    hip_rt.synchronize()
    got = c.d_weight.numpy().astype(np.float64)
    for b, L in enumerate(c.lens):
        # lse and weights each off by (D + keys + 64) steps of the largest score at most
        bound = Hq // G * (4 * D + 2 * L + 64) * C.U32 * 4
        assert np.abs(got[b, :, :L + 1].sum(-1) - Hq // G).max() <= bound * (Hq // G)


def test_nan_reaches_the_weights_that_saw_it(am, dev):
    import hip_rt
    c = Cache(am, "f32", 1, 2, 80, 64, [70])
    k = c.K.host.copy()
    k[0, 0, 13] = np.nan
    c.K.base.upload(c.K._flat(k))
    q = C.Tensor(np.random.default_rng(1).standard_normal((1, 4, 1, 64)), "f32")
    kd = C.Tensor(np.ones((1, 2, 1, 64), np.float32), "f32")
    d = am.Drafts(q.dev, kd.dev, kd.dev)
    am.cache_weigh_ex(c.desc, d, C.floats(np.full((1, 4, 1), 3.0)), weight_in=None)
    hip_rt.synchronize()
    w = c.d_weight.numpy()[0, :, :71]
    assert np.isnan(w[0, 13]) and np.isfinite(np.delete(w[0], 13)).all() and np.isfinite(w[1]).all()


# ---------------------------------------------------------------- eviction
def check_evict(am, c, budget, recent, workspace=None):
    K, V, weight, pos = c.K.numpy(), c.V.numpy(), c.d_weight.numpy(), c.d_pos.numpy()
    want = [x.copy() for x in (K, V, weight, pos)]
    moves = 0
    B, G = c.shape[:2]
    for b in range(B):
        for g in range(G):
            for to, frm in C.evict_moves(weight[b, g], pos[b, g], c.lens[b], c.seen[b], budget,
                                         recent):
                for x, y in zip(want, (K, V, weight, pos)):
                    x[b, g, to] = y[b, g, frm]
                moves += 1
    am.cache_evict_ex(c.desc, budget, recent, workspace)
    c.same(*want)
    assert c.d_len.numpy().tolist() == c.lens
    return moves


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cap,budget,recent,lens", [
    (1, 1, 1, [1]), (2, 1, 0, [2, 1]), (5, 4, 4, [5, 5]), (64, 32, 0, [64, 63]),
    (65, 64, 10, [65, 64]), (100, 7, 3, [100, 0]), (300, 299, 1, [300, 299]),
    (1000, 500, 100, [999, 750]), (1500, 1, 1, [1025, 1024]), (4097, 2000, 2000, [4097, 3000]),
    (9000, 8000, 64, [9000, 8001]),
    (16385, 9000, 300, [16385, 16384]), (40000, 11111, 4000, [40000, 20000])])
def test_evict(am, dev, dtype, cap, budget, recent, lens):
    print(f"[case] evict {dtype} {cap} {budget} {recent} {lens}", flush=True)
    c = Cache(am, dtype, len(lens), 2, cap, 24, lens, seen=[cap] * len(lens), seed=cap)
    check_evict(am, c, budget, recent)


@pytest.mark.parametrize("D,order,offset,pad", [(1, "heads", 0, 0), (77, "rows", 0, 1),
                                                (128, "rows", 8, 8), (512, "heads", 1, 0),
                                                (8192, "heads", 0, 0)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_evict_layouts(am, dev, dtype, D, order, offset, pad):
    c = Cache(am, dtype, 2, 3, 150, D, [150, 140], seen=[150] * 2, order=order, offset=offset,
              pad=pad, fill=np.nan)
    assert check_evict(am, c, 90, 20) > 0


@pytest.mark.parametrize("kind", ["equal", "zeros", "two", "infinite", "nan", "all nan", "negative",
                                  "tiny", "digits"])
def test_evict_ranks(am, dev, kind):
    """Ties go to the lower row; NaN ranks below everything, -0 as 0."""
    import hip_rt
    B, G, cap, L = 2, 2, 700, 650
    c = Cache(am, "bf16", B, G, cap, 8, [L, L - 7], seen=[cap] * 2)
    rng = np.random.default_rng(7)
    w = {"equal": lambda: np.full((B, G, cap), 0.25),
         "zeros": lambda: np.where(rng.random((B, G, cap)) < 0.5, 0.0, -0.0),
         "two": lambda: rng.integers(0, 2, (B, G, cap)) * 1.5,
         "infinite": lambda: rng.choice([np.inf, -np.inf, 1.0, 0.0], (B, G, cap)),
         "nan": lambda: rng.choice([np.nan, -np.nan, -np.inf, 1.0, 2.0], (B, G, cap)),
         "all nan": lambda: np.full((B, G, cap), np.nan),
         "negative": lambda: rng.standard_normal((B, G, cap)),
         "tiny": lambda: rng.integers(0, 40, (B, G, cap)) * 1e-45,
         "digits": lambda: (rng.integers(0, 4, (B, G, cap)) + 0x3f800000).astype(np.uint32)
         .view(np.float32).reshape(B, G, cap)}[kind]()
    c.d_weight.upload(w.astype(np.float32))
    for budget, recent in ((300, 50), (300, 0)):
        assert check_evict(am, c, budget, recent) > 0 or kind in ("equal", "zeros", "all nan")
        c.d_weight.upload(w.astype(np.float32))


@pytest.mark.parametrize("seen,recent,dup", [(700, 0, 0), (700, 120, 0), (10, 5, 0), (1 << 30, 300, 0),
                                             (-(1 << 31), 300, 0), (700, 300, 1)])
def test_evict_recent(am, dev, seen, recent, dup):
    """Positions decide what is recent; more recent rows than the budget holds keep the lower ones."""
    c = Cache(am, "f32", 1, 3, 700, 4, [700], seen=[seen])
    if dup:
        c.pos[...] = np.where(c.pos % 2, 699, c.pos)
        c.d_pos.upload(c.pos)
    check_evict(am, c, 300, recent)


def test_evict_workspace(am, dev):
    import hip_rt
    c = Cache(am, "bf16", 2, 2, 500, 16, [500, 400], seen=[500] * 2)
    n = am.cache_evict_workspace_bytes(c.desc, 200)
    ws = hip_rt.DeviceArray((n // 4 + 64,), "i32", fill=0x5A)
    mine = hip_rt.DeviceArray.wrap(ws.ptr, (n // 4,), "i32", keep=ws)
    check_evict(am, c, 200, 20, mine)
    words = ws.numpy()
    assert (words[:40960 // 4] == 0x5A5A5A5A).all() and (words[n // 4:] == 0x5A5A5A5A).all()


def test_evict_captured(am, dev):
    """A captured eviction replayed with other lengths and weights."""
    import hip_rt
    s = hip_rt.Stream()
    c = Cache(am, "bf16", 2, 2, 600, 32, [600, 10], seen=[600] * 2)
    call = am.cache_evict_call(c.desc, 256, 30)
    call(s)
    s.synchronize()
    g = hip_rt.Graph(s, lambda: call(s))
    rng = np.random.default_rng(1)
    for lens in ([300, 600], [256, 257], [0, 599], [600, 600]):
        c.lens = lens
        c.d_len.upload(np.array(lens, np.int32))
        w = rng.random(c.weight.shape).astype(np.float32)
        c.d_weight.upload(w)
        K, V, pos = c.K.numpy(), c.V.numpy(), c.d_pos.numpy()
        want = [x.copy() for x in (K, V, w, pos)]
        for b in range(2):
            for h in range(2):
                for to, frm in C.evict_moves(w[b, h], pos[b, h], lens[b], 600, 256, 30):
                    for x, y in zip(want, (K, V, w, pos)):
                        x[b, h, to] = y[b, h, frm]
        g.launch()
        s.synchronize()
        c.same(*want)
        am.cache_advance_ex(c.desc, limit=600, stream=s)  # eager work between replays
    g.destroy()
    s.destroy()


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("dtype,D,Hq,G", [("bf16", 128, 8, 2), ("f32", 64, 4, 4), ("bf16", 520, 4, 2)])
@pytest.mark.parametrize("captured", [False, True])
def test_decoding(am, dev, dtype, D, Hq, G, captured):
    """Steps of a decoding program for two layers that share their lengths: attention of a tree
    of drafts, commit of a path, weights, lengths, and eviction over the bound; against the same
    program on the host in float64."""
    import hip_rt
    B, T, cap, budget, recent = 3, 6, 80, 48, 12
    s = hip_rt.Stream()
    rng = np.random.default_rng(11)
    layers = [Cache(am, dtype, B, G, cap, D, [40, 0, 47], seed=i) for i in range(2)]
    first = layers[0]
    lens, seen = list(first.lens), list(first.seen)
    for c in layers[1:]:
        c.desc = am.KvCache(c.K.dev, c.V.dev, first.d_len, first.d_seen, c.d_weight, c.d_pos)
    host = [dict(K=c.K.host.copy(), V=c.V.host.copy(), w=c.weight.astype(np.float64),
                 pos=c.pos.copy()) for c in layers]
    steps = []
    for c in layers:
        t = dict(zip("qkv", (C.Tensor(np.zeros((B, h, T, D)), dtype) for h in (Hq, G, G))))
        t["out"], t["lse"] = C.Tensor(np.zeros((B, Hq, T, D)), dtype), C.floats(np.zeros((B, Hq, T)))
        steps.append(t)
    count, mask = C.ints([T] * B), C.ints(np.zeros((B, T, 1)))
    path, accepted = C.ints(np.zeros((B, 4))), C.ints([0] * B)
    attend, settle, cut = [], [], []
    for c, t in zip(layers, steps):
        d = am.Drafts(t["q"].dev, t["k"].dev, t["v"].dev, count=count, mask=mask)
        attend.append(am.tree_attention_call(c.desc, d, t["out"].dev, t["lse"]))
        settle.append(am.cache_commit_call(c.desc, d, path, accepted))
        settle.append(am.cache_weigh_call(c.desc, d, t["lse"], path, accepted))
        cut.append(am.cache_evict_call(c.desc, budget, recent))
    settle.append(am.cache_advance_call(first.desc, d, path, accepted))
    cut.append(am.cache_advance_call(first.desc, limit=budget))

    def both():
        for call in attend:
            call(s)

    def after():
        for call in settle + cut:
            call(s)

    for call in cut[:-1] + attend:  # workspaces
        call(s)
    s.synchronize()
    for c, h in zip(layers, host):  # (nothing over the bound yet: no change)
        assert np.array_equal(c.d_pos.numpy(), h["pos"])
    graphs = [hip_rt.Graph(s, both), hip_rt.Graph(s, after)] if captured else None
    for step in range(6):
        counts = [int(rng.integers(1, T + 1)) for _ in range(B)]
        parents = [[int(rng.integers(-1, t)) if t else -1 for t in range(T)] for _ in range(B)]
        words = am.tree_mask(parents)
        count.upload(np.array(counts, np.int32))
        mask.upload(words)
        for t in steps:
            for x, h in (("q", Hq), ("k", G), ("v", G)):
                t[x].host = C.rounded(rng.standard_normal((B, h, T, D)) * (2 if x == "q" else 1), dtype)
                t[x].base.upload(t[x]._flat(t[x].host))
        graphs[0].launch() if captured else both()
        s.synchronize()
        # a path from a leaf up to its root
        paths, acc = np.full((B, 4), -1), []
        for b in range(B):
            t, up = counts[b] - 1, []
            while t >= 0:
                up.append(t)
                t = parents[b][t]
            up = up[::-1][:4]
            paths[b, :len(up)] = up
            acc.append(len(up))
        path.upload(paths.astype(np.int32))
        accepted.upload(np.array(acc, np.int32))
        for c, t, h in zip(layers, steps, host):
            want, want_lse, info = C.attend64(t["q"].host, h["K"], h["V"], t["k"].host, t["v"].host,
                                              lens, counts, words)
            C.attend_close(dtype, D, t["out"].numpy(), t["lse"].numpy(), want, want_lse, info, counts)
        graphs[1].launch() if captured else after()
        s.synchronize()
        rows = C.accepted_rows(paths.tolist(), acc, counts, lens, cap, 4)
        new_lens = [l + r for l, r in zip(lens, rows)]
        for c, t, h in zip(layers, steps, host):
            for b in range(B):
                for i in range(rows[b]):
                    r = lens[b] + i
                    h["K"][b, :, r] = t["k"].host[b, :, paths[b][i]]
                    h["V"][b, :, r] = t["v"].host[b, :, paths[b][i]]
                    h["w"][b, :, r], h["pos"][b, :, r] = 0, seen[b] + i
            add, err = weigh64(t["q"].host, h["K"], t["lse"].numpy(), paths.tolist(), rows, lens,
                               1.0 / np.sqrt(D))
            h["w"] += add
            # the ranking is the device's: weights that differ by less than their error may rank
            # either way, so the moves are taken from the device's weights before the cut
            got_pos, got_K = c.d_pos.numpy(), c.K.numpy()
            for b in range(B):
                if new_lens[b] <= budget:
                    n = new_lens[b]
                    assert np.array_equal(got_pos[b, :, :n], h["pos"][b, :, :n])
                    continue
                for g in range(G):
                    at = {row.tobytes(): r for r, row in enumerate(h["K"][b, g, :new_lens[b]])}
                    src = [at[row.tobytes()] for row in got_K[b, g, :budget]]
                    assert np.array_equal(got_pos[b, g, :budget], h["pos"][b, g, src])
                    assert len(set(src)) == budget
                    # rows below the bound stay; what was dropped weighs no more than what was kept
                    assert all(x == r or x >= budget for r, x in enumerate(src))
                    gone = sorted(set(range(new_lens[b])) - set(src))
                    since = seen[b] + rows[b] - recent
                    assert all(h["pos"][b, g, r] < since for r in gone)
                    old = [r for r in src if h["pos"][b, g, r] < since]
                    tol = (err[b, g] + 100 * C.U32 * h["w"][b, g]).max() * 2 * (step + 1)
                    assert not old or h["w"][b, g, gone].max() <= h["w"][b, g, old].min() + tol
                    for x in ("K", "V", "w", "pos"):
                        h[x][b, g, :budget] = h[x][b, g, src].copy()
            lim = [min(l, budget) for l in new_lens]
            got_w = c.d_weight.numpy()
            for b in range(B):
                n = lim[b]
                assert np.array_equal(c.K.numpy()[b, :, :n], h["K"][b, :, :n])
                assert np.array_equal(c.V.numpy()[b, :, :n], h["V"][b, :, :n])
                assert np.abs(got_w[b, :, :n] - h["w"][b, :, :n]).max() <= \
                    (step + 1) * ((err.max() + 100 * C.U32 * max(1.0, h["w"].max())))
        lens = [min(l, budget) for l in new_lens]
        seen = [x + r for x, r in zip(seen, rows)]
        assert first.d_len.numpy().tolist() == lens and first.d_seen.numpy().tolist() == seen
    for g in graphs or []:
        g.destroy()
    s.destroy()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,offset", [(1, 0), (24, 0), (128, 0), (100, 1)])
@pytest.mark.parametrize("cap,budget,recent,lens", [
    (70, 64, 16, [70, 69]), (2000, 1990, 100, [2000, 1991]), (5000, 4960, 64, [5000, 4961]),
    (40000, 39990, 500, [40000, 39995])])
def test_evict_little_over_the_bound(am, dev, dtype, D, offset, cap, budget, recent, lens):
    """Few moves a head, of caches of every size."""
    print(f"[case] evict few {dtype} {D} {cap} {budget} {lens}", flush=True)
    c = Cache(am, dtype, 2, 2, cap, D, lens, seen=[cap] * 2, offset=offset, seed=cap)
    check_evict(am, c, budget, recent)
