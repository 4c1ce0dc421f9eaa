"""Attention of drafted tokens over a key/value cache on the GPU, against the definition in
float64: sizes that fit no tile, lengths from zero, masks that leave tokens nothing, anything
in places that no token attends, strides and alignments, streams and captured graphs."""
import numpy as np
import pytest

import cache_helpers as C
import helpers as H

pytestmark = pytest.mark.gpu


def tree_words(am, rng, B, T):
    return am.tree_mask([[int(rng.integers(-1, t)) if t else -1 for t in range(T)]
                         for _ in range(B)])


def random_words(rng, B, T, keep=0.4):
    """Any visibility; the first draft of each sequence attends no draft."""
    see = np.zeros((B, T, (T + 31) // 32 * 32), bool)
    see[:, 1:, :T] = rng.random((B, T - 1, T)) < keep
    return np.packbits(see, axis=-1, bitorder="little").view("<i4")


class Problem:
    def __init__(self, am, dtype, B, Hq, G, T, D, cap, lens, counts=None, mask="chain",
                 order="heads", offset=0, pad=0, seed=1, sigma=1.5, drafts=True, fill=None):
        rng = np.random.default_rng(seed)
        self.am, self.dtype, self.D, self.lens = am, dtype, D, lens
        self.counts = [T] * B if counts is None else counts

        def make(heads, rows, s=1.0):
            return rng.standard_normal((B, heads, rows, D)).astype(np.float32) * np.float32(s)

        q, k, v, kd, vd = (make(Hq, T, sigma), make(G, cap), make(G, cap), make(G, T), make(G, T))
        if fill is not None:  # in everything that no token may attend
            for b in range(B):
                k[b, :, lens[b]:] = fill
                v[b, :, lens[b]:] = fill
                for x in (q, kd, vd):
                    x[b, :, self.counts[b]:] = fill
        self.words = {"chain": lambda: None, "tree": lambda: tree_words(am, rng, B, T),
                      "random": lambda: random_words(rng, B, T)}[mask]()
        lay = dict(order=order, offset=offset, pad=pad)
        self.Q, self.K, self.V = (C.Tensor(x, dtype, **lay) for x in (q, k, v))
        self.Kd, self.Vd = (C.Tensor(x, dtype, **lay) if drafts else None for x in (kd, vd))
        self.out = C.Tensor(np.full(q.shape, 7.0, np.float32), dtype, **lay)
        self.lse = C.floats(np.full((B, Hq, T), 7.0))
        self.len = C.ints(lens)
        self.cache = am.KvCache(self.K.dev, self.V.dev, self.len)
        self.drafts = am.Drafts(self.Q.dev, self.Kd.dev if drafts else None,
                                self.Vd.dev if drafts else None,
                                count=None if counts is None else C.ints(counts),
                                mask=None if self.words is None else C.ints(self.words))

    def want(self, lens=None, scale=None):
        return C.attend64(self.Q.host, self.K.host, self.V.host,
                          None if self.Kd is None else self.Kd.host,
                          None if self.Vd is None else self.Vd.host,
                          self.lens if lens is None else lens, self.counts, self.words, scale)

    def check(self, lens=None, scale=None):
        out, lse = self.out.numpy(), self.lse.numpy()
        want, want_lse, info = self.want(lens, scale)
        C.attend_close(self.dtype, self.D, out, lse, want, want_lse, info, self.counts)
        for b, n in enumerate(self.counts):  # rows behind the last token
            assert (out[b, :, n:] == 7.0).all() and (lse[b, :, n:] == 7.0).all()

    def run(self, scale=0.0, max_len=0, workspace=None, stream=None):
        import hip_rt
        self.am.tree_attention_ex(self.cache, self.drafts, self.out.dev, self.lse, scale, max_len,
                                  workspace, stream)
        hip_rt.synchronize()


def solve(am, dtype, B, Hq, G, T, D, cap, lens, **kw):
    print(f"[case] tree attention {dtype} {(B, Hq, G, T, D, cap)} len={lens} {kw}", flush=True)
    p = Problem(am, dtype, B, Hq, G, T, D, cap, lens, **kw)
    p.run()
    p.check()


DIMS = [1, 3, 8, 20, 64, 65, 80, 96, 100, 128, 130, 160, 192, 200, 256, 257, 264, 384, 500, 512,
        1000, 1024, 2048, 4100, 8192]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", DIMS)
def test_head_sizes(am, dev, dtype, D):
    solve(am, dtype, 2, 4, 2, 3, D, 90, [77, 33], mask="tree", seed=D)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 512])
@pytest.mark.parametrize("L", [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256,
                               257, 511, 513, 1023, 1025])
def test_lengths_single_token(am, dev, dtype, D, L):
    solve(am, dtype, 1, 2, 1, 1, D, max(L, 1), [L], seed=L)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T", [1, 2, 5, 8, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 129, 256])
@pytest.mark.parametrize("mask", ["chain", "tree", "random"])
def test_draft_counts(am, dev, dtype, T, mask):
    solve(am, dtype, 2, 2, 1, T, 64, 50, [50, 0], counts=[T, max(1, T - 3)], mask=mask, seed=T)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("Hq,G", [(1, 1), (3, 3), (8, 1), (6, 2), (10, 2), (32, 4), (71, 1)])
@pytest.mark.parametrize("D", [128, 640])
def test_shared_heads(am, dev, dtype, Hq, G, D):
    solve(am, dtype, 2, Hq, G, 5, D, 200, [140, 61], mask="tree", seed=Hq)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [72, 128, 520])
@pytest.mark.parametrize("order", ["heads", "rows"])
@pytest.mark.parametrize("offset,pad", [(0, 0), (1, 0), (0, 3), (8, 8), (2, 1), (4, 4)])
def test_strides_and_alignment(am, dev, dtype, D, order, offset, pad):
    solve(am, dtype, 2, 4, 2, 6, D, 70, [70, 41], mask="tree", order=order, offset=offset, pad=pad)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fill", [np.nan, np.inf, -np.inf, 3e38])
@pytest.mark.parametrize("D", [48, 128, 300])
@pytest.mark.parametrize("L", [0, 40, 64])
def test_anything_where_no_token_looks(am, dev, dtype, fill, D, L):
    """Rows past the length, drafts past the count and their queries."""
    solve(am, dtype, 2, 4, 2, 20, D, 100, [L, 37], counts=[13, 20], mask="random", fill=fill)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fill", [np.nan, np.inf])
@pytest.mark.parametrize("D,T", [(128, 9), (256, 40), (520, 9)])
def test_masked_draft_of_anything(am, dev, dtype, fill, D, T):
    """A draft that some tokens attend and others do not: only those that do may see its values."""
    import hip_rt
    print(f"[case] masked draft {dtype} {fill} {D} {T}", flush=True)
    p = Problem(am, dtype, 2, 4, 2, T, D, 50, [50, 0], mask="tree", seed=9)
    bad = T // 2
    kd, vd = p.Kd.host.copy(), p.Vd.host.copy()
    kd[:, :, bad] = np.nan if np.isnan(fill) else kd[:, :, bad]
    vd[:, :, bad] = fill
    p.Kd.base.upload(p.Kd._flat(kd))
    p.Vd.base.upload(p.Vd._flat(vd))
    p.run()
    want, want_lse, info = p.want()
    out, lse = p.out.numpy(), p.lse.numpy()
    for b in range(2):
        see = C.visible(T, T, p.words, b)[:, bad]
        assert see.any() and not see.all()
        one = [x[b:b + 1][:, :, ~see] for x in (out, lse, want, want_lse)]
        inf1 = {k: x[b:b + 1][:, :, ~see] for k, x in info.items()}
        C.attend_close(dtype, D, *one, inf1, [int((~see).sum())])
        assert not np.isfinite(out[b][:, see]).any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [128, 512])
def test_nothing_to_attend(am, dev, dtype, D):
    """No rows in use and no draft visible: zeros and -infinity."""
    import hip_rt
    p = Problem(am, dtype, 2, 2, 2, 4, D, 8, [0, 0], mask="random", fill=np.nan)
    p.drafts = am.Drafts(p.Q.dev, p.Kd.dev, p.Vd.dev, mask=C.ints(np.zeros((2, 4, 1))))
    p.run()
    assert (p.out.numpy() == 0).all() and np.isneginf(p.lse.numpy()).all()
    # the same without any draft keys
    p = Problem(am, dtype, 2, 2, 2, 4, D, 8, [0, 5], drafts=False)
    p.run()
    p.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 256, 1024])
def test_without_draft_keys(am, dev, dtype, D):
    """Queries of several tokens over padded states, no keys of their own."""
    solve(am, dtype, 3, 8, 2, 6, D, 150, [150, 0, 77], counts=[6, 6, 2], drafts=False)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [128, 520])
@pytest.mark.parametrize("case", ["nan", "inf", "overflow"])
def test_scores_without_a_number(am, dev, dtype, D, case):
    """NaN in an attended key is NaN in the output; scores of -infinity alone are nothing to
    attend; one score of -infinity has weight zero."""
    p = Problem(am, dtype, 1, 2, 2, 3, D, 40, [40], drafts=False, seed=4)
    q, k = p.Q.host.copy(), p.K.host.copy()
    q[...] = np.abs(q)
    if case == "nan":
        k[0, 0, 11] = np.nan
    elif case == "inf":
        k[0, 0, :] = -np.inf
    else:
        k[0, 0, 17] = -np.inf
    p.Q.base.upload(p.Q._flat(q))
    p.K.base.upload(p.K._flat(k))
    p.run()
    out, lse = p.out.numpy(), p.lse.numpy()
    q, k, v = C.rounded(q, dtype), C.rounded(k, dtype), p.V.host
    if case == "nan":
        assert np.isnan(out[0, 0]).all() and np.isfinite(out[0, 1]).all()
    elif case == "inf":
        assert (out[0, 0] == 0).all() and np.isneginf(lse[0, 0]).all()
    else:
        k2, v2 = np.delete(k, 17, 2), np.delete(v, 17, 2)
        want, want_lse, info = C.attend64(q, k2, v2, None, None, [39], [3])
        C.attend_close(dtype, D, out[:, :1], lse[:, :1], want[:, :1], want_lse[:, :1],
                       {x: y[:, :1] for x, y in info.items()}, [3])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [0.03, 4.0, -0.5])
@pytest.mark.parametrize("D", [96, 512])
def test_scale(am, dev, dtype, scale, D):
    scale = float(np.float32(scale))
    p = Problem(am, dtype, 1, 4, 2, 5, D, 300, [300], mask="tree", sigma=2.0)
    p.run(scale=scale)
    p.check(scale=scale)


@pytest.mark.parametrize("dtype,Hq,G,T,D,L", [
    ("bf16", 8, 2, 16, 128, 6000), ("f32", 4, 2, 4, 128, 5001), ("bf16", 4, 4, 1, 64, 12345),
    ("bf16", 4, 1, 33, 256, 3001), ("f32", 2, 2, 2, 512, 2500), ("bf16", 2, 1, 3, 1024, 4099),
    ("bf16", 16, 2, 64, 96, 2049)])
def test_long_caches(am, dev, dtype, Hq, G, T, D, L):
    solve(am, dtype, 1, Hq, G, T, D, L + 9, [L], mask="tree", seed=L)


def test_lengths_out_of_range_are_clamped(am, dev):
    p = Problem(am, "bf16", 3, 4, 2, 4, 128, 60, [60, 0, 30], counts=[4, 4, 4])
    p.len.upload(np.array([1 << 30, -5, 30], np.int32))
    p.drafts.count.upload(np.array([99, 4, -1], np.int32))
    p.counts = [4, 4, 0]
    p.run()
    p.check()


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f32", 128), ("bf16", 640)])
def test_max_len_bounds_the_lengths(am, dev, dtype, D):
    p = Problem(am, dtype, 2, 4, 2, 5, D, 1500, [1500, 700], mask="tree")
    for max_len in (1, 100, 701, 1499, 1500, 1 << 30):
        p.run(max_len=max_len)
        p.check(lens=[min(l, max_len) for l in p.lens])


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f32", 96), ("bf16", 520)])
def test_workspaces(am, dev, dtype, D):
    """A caller's workspace of the size asked for, with the words in front left alone and nothing
    behind it touched; the library's gives the same bits."""
    import hip_rt
    p = Problem(am, dtype, 1, 4, 2, 5, D, 2000, [1999], mask="tree")
    n = am.tree_attention_workspace_bytes(p.cache, p.drafts)
    assert n >= 40960 and n % 4 == 0
    ws = hip_rt.DeviceArray((n // 4 + 64,), "i32", fill=0x5A)
    mine = hip_rt.DeviceArray.wrap(ws.ptr, (n // 4,), "i32", keep=ws)
    p.run(workspace=mine)
    p.check()
    words = ws.numpy()
    assert (words[:40960 // 4] == 0x5A5A5A5A).all() and (words[n // 4:] == 0x5A5A5A5A).all()
    first = p.out.base.bits()
    p.run()
    assert np.array_equal(first, p.out.base.bits())


@pytest.mark.parametrize("dtype,Hq,G,T,D", [("bf16", 8, 2, 3, 128), ("f32", 4, 2, 2, 64),
                                            ("bf16", 2, 1, 4, 600), ("bf16", 16, 2, 40, 128)])
def test_captured_calls_follow_the_lengths(am, dev, dtype, Hq, G, T, D):
    """A captured call replayed with other lengths, counts and masks, with eager calls between."""
    import hip_rt
    s = hip_rt.Stream()
    p = Problem(am, dtype, 2, Hq, G, T, D, 900, [500, 20], counts=[T, T], mask="tree", seed=3)
    p.run(stream=s)  # the stream's workspace
    call = am.tree_attention_call(p.cache, p.drafts, p.out.dev, p.lse)
    graph = hip_rt.Graph(s, lambda: call(s))
    rng = np.random.default_rng(0)
    for lens in ([900, 1], [0, 333], [64, 65], [500, 899]):
        counts = [int(rng.integers(1, T + 1)), T]
        p.len.upload(np.array(lens, np.int32))
        p.drafts.count.upload(np.array(counts, np.int32))
        p.words = tree_words(am, rng, 2, T)
        p.drafts.mask.upload(p.words)
        p.out.base.upload(p.out._flat(np.full(p.out.host.shape, 7.0, np.float32)))
        p.lse.upload(np.full(p.lse.shape, 7.0, np.float32))
        p.counts = counts
        graph.launch()
        s.synchronize()
        p.check(lens=lens)
        graph_bits = p.out.base.bits()
        p.run(stream=s)
        assert np.array_equal(graph_bits, p.out.base.bits())
    graph.destroy()
    s.destroy()


def test_capture_refuses_to_allocate(am, dev):
    import hip_rt
    s = hip_rt.Stream()
    # (more scratch than the workspace of any stream of the other tests, whose handle this one
    # may have)
    p = Problem(am, "bf16", 1, 32, 8, 64, 128, 4096, [4000])
    assert am.tree_attention_workspace_bytes(p.cache, p.drafts) > 8 << 20
    status = []

    def call():
        try:
            am.tree_attention_ex(p.cache, p.drafts, p.out.dev, p.lse, stream=s)
        except am.AtnError as e:
            status.append(e.status)

    hip_rt.Graph(s, call).destroy()
    assert status == [am.ATN_ERR_CAPTURE]
    p.run(stream=s)
    p.check()
    s.destroy()


def test_two_streams_at_once(am, dev):
    """Calls on two streams, each with the stream's own scratch."""
    import hip_rt
    ps = [Problem(am, "bf16", 2, 8, 2, 4, 128, 4000, [4000, 2500], mask="tree", seed=i)
          for i in range(2)]
    ss = [hip_rt.Stream() for _ in ps]
    for _ in range(3):
        for p, s in zip(ps, ss):
            am.tree_attention_ex(p.cache, p.drafts, p.out.dev, p.lse, stream=s)
    hip_rt.synchronize()
    for p in ps:
        p.check()
    for s in ss:
        s.destroy()


def test_same_bits_every_time(am, dev):
    p = Problem(am, "bf16", 4, 16, 4, 9, 128, 3000, [3000, 100, 0, 1777], mask="tree")
    p.run()
    first = p.out.base.bits()
    for _ in range(5):
        p.run()
        assert np.array_equal(first, p.out.base.bits())


def test_cache_past_32_bit_offsets(am, dev):
    """Rows whose element offsets in a head pass 2^31: a cache of few rows far apart."""
    import hip_rt
    D, cap, ld = 128, 40, 1 << 26  # the last row starts 39 * 2^26 elements in
    rng = np.random.default_rng(5)
    kv = rng.standard_normal((2, cap, D)).astype(np.float32)
    big = hip_rt.DeviceArray(((cap - 1) * ld + 2 * D,), "bf16")
    for r in range(cap):
        row = hip_rt.DeviceArray.view(big, r * ld, (2, D))
        row.upload(kv[:, r])
    q = C.Tensor(rng.standard_normal((1, 4, 2, D)), "bf16")
    K = hip_rt.DeviceArray.wrap(big.ptr, (1, 1, cap, D), "bf16", strides=(0, 0, ld, 1), keep=big)
    V = hip_rt.DeviceArray.wrap(big.ptr + 2 * D, (1, 1, cap, D), "bf16", strides=(0, 0, ld, 1),
                                keep=big)
    out, lse = C.Tensor(np.zeros((1, 4, 2, D)), "bf16"), C.floats(np.zeros((1, 4, 2)))
    print("[case] rows 2^26 elements apart", flush=True)
    am.tree_attention_ex(am.KvCache(K, V, C.ints([cap])), am.Drafts(q.dev), out.dev, lse)
    hip_rt.synchronize()
    k, v = (C.rounded(x, "bf16")[None, None] for x in kv)
    want, want_lse, info = C.attend64(q.host, k, v, None, None, [cap], [2])
    C.attend_close("bf16", D, out.numpy(), lse.numpy(), want, want_lse, info, [2])
    big.free()


# ---------------------------------------------------------------- many sequences, many rows
def many_lens(rng, B, cap):
    """Mostly short, some empty, a few to the capacity."""
    lens = rng.integers(0, 40, B)
    lens[rng.random(B) < 0.2] = 0
    lens[rng.integers(0, B, 5)] = cap
    lens[rng.integers(0, B, 5)] = rng.integers(1, cap, 5)
    return [int(x) for x in lens]


@pytest.mark.parametrize("dtype,Hq,G,T,D,cap", [
    ("bf16", 4, 2, 2, 128, 1300), ("f32", 2, 2, 1, 72, 700), ("bf16", 2, 1, 3, 520, 400),
    ("bf16", 2, 1, 3, 264, 1100), ("bf16", 6, 1, 20, 100, 1100)])
@pytest.mark.parametrize("B", [63, 64, 65, 128, 131])
def test_many_sequences(am, dev, dtype, Hq, G, T, D, cap, B):
    """More sequences than a wave has lanes."""
    rng = np.random.default_rng(B)
    counts = [int(x) for x in rng.integers(0, T + 1, B)]
    solve(am, dtype, B, Hq, G, T, D, cap, many_lens(rng, B, cap), counts=counts, mask="tree", seed=B)


@pytest.mark.parametrize("Hq,G,T,D,lens,mask", [
    (65, 1, 1, 128, [700, 64], "chain"), (4, 2, 50, 128, [333, 0], "random"),
    (4, 1, 33, 96, [100, 1500], "tree"), (2, 1, 150, 65, [31, 97], "random"),
    (4, 1, 150, 128, [64, 2000], "tree"), (8, 2, 256, 128, [40, 257], "random"),
    (13, 1, 100, 120, [1, 640], "random"), (3, 1, 256, 100, [3000, 77], "tree")])
@pytest.mark.parametrize("layout", [{}, dict(order="rows", offset=3, pad=5)])
def test_many_rows(am, dev, Hq, G, T, D, lens, mask, layout):
    """More than 64 query rows of a kv head, of one to several tiles, and NaN where none may look."""
    solve(am, "bf16", 2, Hq, G, T, D, max(lens) + 40, lens, counts=[T, T - T // 3], mask=mask,
          fill=np.nan, seed=T, **layout)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("Hq,T,D", [(2, 100, 64), (2, 100, 24), (5, 40, 192), (3, 70, 256),
                                    (2, 90, 640)])
def test_several_row_tiles(am, dev, dtype, Hq, T, D):
    solve(am, dtype, 2, Hq, 1, T, D, 500, [460, 131], counts=[T - 9, T], mask="random", fill=np.nan,
          seed=T)


@pytest.mark.parametrize("fill", [np.nan, np.inf])
@pytest.mark.parametrize("lens", [[50, 0], [64, 3000]])
def test_masked_draft_of_anything_many_rows(am, dev, fill, lens):
    T, D, bad = 60, 128, 31
    print(f"[case] masked draft, many rows {fill} {lens}", flush=True)
    p = Problem(am, "bf16", 2, 4, 2, T, D, max(lens), lens, mask="tree", seed=9)
    kd, vd = p.Kd.host.copy(), p.Vd.host.copy()
    kd[:, :, bad] = np.nan if np.isnan(fill) else kd[:, :, bad]
    vd[:, :, bad] = fill
    p.Kd.base.upload(p.Kd._flat(kd))
    p.Vd.base.upload(p.Vd._flat(vd))
    p.run()
    want, want_lse, info = p.want()
    out, lse = p.out.numpy(), p.lse.numpy()
    for b in range(2):
        see = C.visible(T, T, p.words, b)[:, bad]
        assert see.any() and not see.all()
        one = [x[b:b + 1][:, :, ~see] for x in (out, lse, want, want_lse)]
        inf1 = {k: x[b:b + 1][:, :, ~see] for k, x in info.items()}
        C.attend_close("bf16", D, *one, inf1, [int((~see).sum())])
        assert not np.isfinite(out[b][:, see]).any()


@pytest.mark.parametrize("Hq,T", [(2, 4), (4, 40)])
def test_nothing_to_attend_many_heads(am, dev, Hq, T):
    """Tokens whose mask is empty beside others', over an empty cache."""
    B, D = 2, 128
    p = Problem(am, "bf16", B, Hq, 1, T, D, 8, [0, 0], mask="random", fill=np.nan, seed=2)
    p.words = p.words.copy()
    p.words[0, ::2] = 0
    p.words[1] = 0
    p.drafts = am.Drafts(p.Q.dev, p.Kd.dev, p.Vd.dev, mask=C.ints(p.words))
    p.run()
    p.check()
    assert (p.out.numpy()[1] == 0).all() and np.isneginf(p.lse.numpy()[1]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,Hq,T", [(48, 2, 3), (128, 2, 3), (128, 4, 40), (200, 2, 20), (300, 2, 3)])
@pytest.mark.parametrize("L", [41, 64, 3000, 3001])
def test_infinite_values(am, dev, dtype, D, Hq, T, L):
    """Infinities in a row of V that all tokens attend, the cache's last: infinite in its dims,
    of their sign, NaN where two of them disagree; the other dims as if it were not there."""
    print(f"[case] infinite values {dtype} {D} {Hq} {T} {L}", flush=True)
    p = Problem(am, dtype, 1, Hq, 1, T, D, L + 3, [L], mask="tree", sigma=0.3, seed=6)
    v = p.V.host.copy()
    v[0, 0, L - 1, 5], v[0, 0, L - 1, 11] = np.inf, -np.inf
    v[0, 0, L - 1, 23], v[0, 0, L - 2, 23] = np.inf, -np.inf
    p.V.base.upload(p.V._flat(v))
    p.run()
    out, lse = p.out.numpy(), p.lse.numpy()
    assert np.isposinf(out[..., 5]).all() and np.isneginf(out[..., 11]).all()
    assert np.isnan(out[..., 23]).all()
    want, want_lse, info = p.want()
    rest = np.delete(np.arange(D), [5, 11, 23])
    info["pv"] = info["pv"][..., rest]
    C.attend_close(dtype, D, out[..., rest], lse, want[..., rest], want_lse, info, [T])


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f32", 72), ("bf16", 520), ("f32", 1100)])
def test_small_workspaces(am, dev, dtype, D):
    """A workspace that holds one pair's scratch: several passes, or fewer ranges; none at all is
    enough where no scores are kept, and refused where they are."""
    import hip_rt
    one = Problem(am, dtype, 1, 2, 1, 5, D, 1500, [1499], mask="tree")
    p = Problem(am, dtype, 3, 6, 3, 5, D, 1500, [1499, 0, 700], mask="tree")
    n = am.tree_attention_workspace_bytes(one.cache, one.drafts)
    assert 40960 < n < am.tree_attention_workspace_bytes(p.cache, p.drafts)
    for size in (n, n + 4096, 2 * n, 3 * n):
        ws = hip_rt.DeviceArray((size // 4 + 64,), "i32", fill=0x5A)
        p.out.base.upload(p.out._flat(np.full(p.out.host.shape, 7.0, np.float32)))
        p.run(workspace=hip_rt.DeviceArray.wrap(ws.ptr, (size // 4,), "i32", keep=ws))
        p.check()
        words = ws.numpy()
        assert (words[:40960 // 4] == 0x5A5A5A5A).all() and (words[size // 4:] == 0x5A5A5A5A).all()
    ws = hip_rt.DeviceArray((40960 // 4,), "i32")
    if D > 256:
        with pytest.raises(am.AtnError) as e:
            p.run(workspace=ws)
        assert e.value.status == am.ATN_ERR_WORKSPACE
    else:
        p.run(workspace=ws)
        p.check()


def test_one_workspace_for_two_graphs(am, dev):
    """Two captured calls of different shapes that share a caller's workspace, replayed in turn."""
    import hip_rt
    s = hip_rt.Stream()
    ps = [Problem(am, "bf16", 2, 8, 2, 3, 128, 3000, [3000, 1200], mask="tree", seed=1),
          Problem(am, "bf16", 1, 2, 1, 4, 600, 1000, [999], mask="tree", seed=2)]
    n = max(am.tree_attention_workspace_bytes(p.cache, p.drafts) for p in ps)
    ws = hip_rt.DeviceArray((n // 4,), "i32", fill=0)
    calls = [am.tree_attention_call(p.cache, p.drafts, p.out.dev, p.lse, workspace=ws) for p in ps]
    graphs = [hip_rt.Graph(s, lambda c=c: c(s)) for c in calls]
    for _ in range(3):
        for p, g in zip(ps, graphs):
            p.out.base.upload(p.out._flat(np.full(p.out.host.shape, 7.0, np.float32)))
            g.launch()
        s.synchronize()
        for p in ps:
            p.check()
        calls[0](s)
        s.synchronize()
    for g in graphs:
        g.destroy()
    s.destroy()
