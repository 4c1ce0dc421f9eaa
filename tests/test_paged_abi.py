"""Rotation and the paged cache, without a GPU: every argument error is reported with its status
before any HIP call, workspace queries, frequencies, the binding's checks, and the kernels' division
by multiplication."""
import ctypes

import numpy as np
import pytest

# device addresses that nothing dereferences
KA, VA, QA, KD, VD, OA, LA, TA, NA, CA, PA, FA, SA, RA = (0x7F0000000000 + i * 0x1000000000
                                                          for i in range(14))


def make(cls, **f):
    x = cls()
    for k, v in f.items():
        setattr(x, k, (ctypes.c_int64 * 3)(*v) if k.endswith("stride") else v)
    return x


def cache(am, **kw):
    return make(am._PagedCacheDesc, **{**dict(K=KA, V=VA, table=TA, len=LA, dtype=1, batch=2,
                                              kv_heads=2, pages=10, page_rows=16, table_pages=4,
                                              head_d=64), **kw})


def drafts(am, **kw):
    return make(am._DraftsDesc, **{**dict(Q=QA, K=KD, V=VD, heads=4, tokens=5, count=CA), **kw})


def rotary(am, **kw):
    return make(am._RotaryDesc, **{**dict(pairing=1, rotary_dim=64, freq=FA, amplitude=1.0), **kw})


def prefix(am, **kw):
    return make(am._SharedPrefixDesc, **{**dict(first=SA, rows=RA, groups=1), **kw})


def ref(x):
    return None if x is None else ctypes.byref(x)


def strides(s):
    return None if s is None else ctypes.cast((ctypes.c_int64 * 3)(*s), ctypes.c_void_p)


def attend(am, c, d, p=None, out=OA, st=None, lse=NA, scale=0.0, max_len=0, ws=None, wsb=0):
    return am.lib().atn_paged_attention_ex(ref(c), ref(d), ref(p), out, strides(st), lse, scale,
                                           max_len, ws, wsb, None)


def append(am, c, d, r=None, pos=None, q_out=OA, st=None):
    return am.lib().atn_paged_append_ex(ref(c), ref(d), ref(r), pos, q_out, strides(st), None)


def advance(am, c, d):
    return am.lib().atn_paged_advance_ex(ref(c), ref(d), None)


def no_device(am):
    """What a call that passes every check gets here."""
    return -6 if am.device_count() < 1 else 0


CALLS = [attend, append, advance]


@pytest.mark.parametrize("op", CALLS)
@pytest.mark.parametrize("kw,code", [
    (dict(dtype=2), -9), (dict(K=None), -1), (dict(V=None), -1), (dict(table=None), -1),
    (dict(len=None), -1), (dict(batch=0), -2), (dict(kv_heads=0), -2), (dict(pages=0), -2),
    (dict(page_rows=0), -2), (dict(table_pages=-1), -2), (dict(head_d=0), -2),
    (dict(head_d=8193), -9), (dict(batch=65536), -4), (dict(page_rows=1 << 20, table_pages=1 << 11), -4),
    (dict(K=KA + 1), -10), (dict(table=TA + 2), -10), (dict(len=LA + 1), -10),
    (dict(k_stride=(-1, 1024, 64)), -9), (dict(v_stride=(2048, 1024, 63)), -9),
    (dict(k_stride=(2048, 64, 64)), -9), (dict(k_stride=(1 << 62, 1024, 64)), -4),
    (dict(v_stride=(64, 640, 1 << 27)), -4)])
def test_cache_refusals(am, op, kw, code):
    assert op(am, cache(am, **kw), drafts(am)) == code


@pytest.mark.parametrize("op", CALLS)
@pytest.mark.parametrize("kw,code", [
    (dict(heads=0), -2), (dict(tokens=0), -2), (dict(heads=5), -9), (dict(tokens=65537), -9),
    (dict(mask=SA), -9), (dict(count=CA + 2), -10), (dict(heads=1 << 17), -4)])
def test_token_refusals(am, op, kw, code):
    assert op(am, cache(am), drafts(am, **kw)) == code


def test_no_descriptors(am):
    for op in CALLS:
        assert op(am, None, drafts(am)) == -1
        assert op(am, cache(am), None) == -1
    assert attend(am, cache(am, batch=256), drafts(am, tokens=40000)) == -4


@pytest.mark.parametrize("kw,code", [
    (dict(d=dict(Q=None)), -1), (dict(out=None), -1), (dict(out=OA + 1), -10), (dict(lse=NA + 2), -10),
    (dict(scale=float("nan")), -9), (dict(scale=float("inf")), -9), (dict(max_len=-1), -2),
    (dict(out=KA), -5), (dict(out=VA + 64), -5), (dict(out=QA), -5), (dict(lse=QA), -5),
    (dict(lse=OA), -5), (dict(out=TA), -5), (dict(lse=LA), -5), (dict(out=CA), -5),
    (dict(st=(0, 64, 256)), -9), (dict(p=dict(groups=0)), -2), (dict(p=dict(groups=3)), -9),
    (dict(p=dict(first=None)), -1), (dict(p=dict(rows=None)), -1), (dict(p=dict(first=SA + 2)), -10),
    (dict(p=dict(), out=SA), -5), (dict(p=dict(), lse=RA), -5),
    (dict(ws=0x1000, wsb=100), -8)])
def test_attention_refusals(am, kw, code):
    kw = dict(kw)
    d, p = kw.pop("d", {}), kw.pop("p", None)
    assert attend(am, cache(am), drafts(am, **d), None if p is None else prefix(am, **p), **kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(d=dict(K=None)), -1), (dict(d=dict(V=None)), -1), (dict(d=dict(Q=None)), -1),
    (dict(r=dict(pairing=2)), -9), (dict(r=dict(rotary_dim=63)), -3), (dict(r=dict(rotary_dim=66)), -3),
    (dict(r=dict(rotary_dim=-2)), -3), (dict(r=dict(freq=None)), -1), (dict(r=dict(freq=FA + 1)), -10),
    (dict(r=dict(amplitude=float("inf"))), -9), (dict(pos=PA + 2), -10), (dict(q_out=OA + 1), -10),
    (dict(q_out=KA), -5), (dict(q_out=KD), -5), (dict(q_out=VD + 128), -5), (dict(q_out=QA + 64), -5),
    (dict(q_out=QA, st=(1280, 64, 256)), -5), (dict(q_out=TA), -5), (dict(q_out=PA, pos=PA), -5),
    (dict(d=dict(K=KA)), -5), (dict(d=dict(V=KA)), -5), (dict(c=dict(V=KA)), -5),
    (dict(c=dict(table=VA)), -5)])
def test_append_refusals(am, kw, code):
    kw = dict(kw)
    c, d, r = (kw.pop(k, {}) for k in "cdr")
    assert append(am, cache(am, **c), drafts(am, **d), rotary(am, **r), **kw) == code


def test_append_in_place_and_without_queries(am):
    ok = no_device(am)
    if ok == 0:
        pytest.skip("addresses that nothing may dereference")
    assert append(am, cache(am), drafts(am), rotary(am), q_out=QA) == ok
    assert append(am, cache(am), drafts(am, Q=None), rotary(am), q_out=None) == ok
    # queries, keys and values as columns of one buffer's rows, the queries turned in place
    row = (4 + 2 + 2) * 64
    s = (5 * row, 64, row)
    d = drafts(am, Q=QA, K=QA + 4 * 128, V=QA + 6 * 128, q_stride=s, k_stride=s, v_stride=s)
    assert append(am, cache(am), d, rotary(am), q_out=QA, st=s) == ok
    # ... but not where the columns meet
    d = drafts(am, Q=QA, K=QA + 4 * 128 - 2, V=QA + 6 * 128, q_stride=s, k_stride=s, v_stride=s)
    assert append(am, cache(am), d, rotary(am), q_out=QA, st=s) == -5


def rotate(am, xs, r, dtype=1, n=None, B=2, T=5, D=64, pos=None, inverse=0):
    a = (am._RotatedDesc * max(1, len(xs)))()
    for i, x in enumerate(xs):
        a[i] = make(am._RotatedDesc, **{**dict(inp=QA, out=OA, heads=4), **x})
    return am.lib().atn_rotary_ex(dtype, ref(r), a, len(xs) if n is None else n, B, T, D, pos, inverse,
                                  None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=3), -9), (dict(n=0), -2), (dict(B=0), -2), (dict(T=0), -2), (dict(D=0), -2),
    (dict(n=4), -9), (dict(D=8193), -9), (dict(B=1 << 12, T=1 << 12), -4), (dict(pos=PA + 1), -10),
    (dict(xs=[dict(inp=None)]), -1), (dict(xs=[dict(out=None)]), -1), (dict(xs=[dict(heads=0)]), -2),
    (dict(xs=[dict(heads=65536)]), -4), (dict(xs=[dict(inp=QA + 1)]), -10),
    (dict(xs=[dict(out=QA + 64)]), -5), (dict(xs=[dict(out=QA, out_stride=(1280, 64, 256))]), -5),
    (dict(xs=[dict(), dict(inp=KD)]), -5), (dict(xs=[dict(), dict(inp=OA, out=VD)]), -5),
    (dict(pos=OA), -5), (dict(xs=[dict(out=FA)]), -5), (dict(xs=[dict(out_stride=(0, 320, 64))]), -9),
    (dict(r=dict(rotary_dim=3)), -3), (dict(r=dict(rotary_dim=128)), -3), (dict(r=dict(freq=None)), -1)])
def test_rotary_refusals(am, kw, code):
    kw = dict(kw)
    xs, r = kw.pop("xs", [dict()]), kw.pop("r", {})
    assert rotate(am, xs, rotary(am, **r), **kw) == code


def test_rotary_without_descriptors(am):
    assert rotate(am, [dict()], None) == -1
    assert am.lib().atn_rotary_ex(1, ref(rotary(am)), None, 1, 2, 5, 64, None, 0, None) == -1


def test_workspace_queries(am):
    def need(c, d, p=None, n=0):
        return am.lib().atn_paged_attention_workspace_bytes(ref(c), ref(d), ref(p), n)

    long = dict(page_rows=64, table_pages=1024, pages=4096, batch=8)
    plain = need(cache(am, **long), drafts(am, tokens=1))
    shared = need(cache(am, **long), drafts(am, tokens=1), prefix(am))
    assert 40960 < plain < shared < 1 << 30
    assert need(cache(am, **long), drafts(am, tokens=1), n=16) == 40960  # whole items: no parts
    assert need(cache(am, **long), drafts(am, mask=SA)) == 0
    assert need(cache(am, **long), drafts(am), prefix(am, groups=9)) == 0
    assert need(None, drafts(am)) == 0 and need(cache(am), None) == 0
    # bounded by fewer kv heads at a time
    big = dict(batch=64, kv_heads=64, pages=1 << 16, page_rows=64, table_pages=1 << 12, head_d=128)
    assert 0 < need(cache(am, **big), drafts(am, heads=64, tokens=512), prefix(am)) <= (1 << 30) + 40960
    # without a prefix a call runs in any workspace; with one a kv head's parts have to fit
    ok = no_device(am)
    if ok != 0:
        assert attend(am, cache(am, **long), drafts(am, tokens=1), ws=0x10000, wsb=40960) == ok
    assert attend(am, cache(am, **long), drafts(am, tokens=1), prefix(am), ws=0x10000, wsb=50000) == -8
    assert attend(am, cache(am, **long), drafts(am, tokens=1), prefix(am), ws=0x10008,
                  wsb=shared) == (-10 if ok == 0 else ok)


@pytest.mark.parametrize("rot", [2, 4, 40, 128])
@pytest.mark.parametrize("base", [10000.0, 500000.0])
def test_frequencies(am, rot, base):
    i = np.arange(rot // 2)
    plain = base ** (-2.0 * i / rot)

    def close(got, want):  # rounded once from fp64, whose powers are off by a few of its steps
        assert got.dtype == np.float32 and got.shape == want.shape
        assert (np.abs(got - want) <= (2.0 ** -24 + 2.0 ** -48) * want).all()

    f, a = am.rope_frequencies(rot, base)
    close(f, plain)
    assert a == 1.0
    f, a = am.rope_frequencies(rot, base, "linear", 8.0)
    close(f, plain / 8)
    f, a = am.rope_frequencies(rot, base, "base", 4.0)
    stretched = plain if rot == 2 else (base * 4.0 ** (rot / (rot - 2))) ** (-2.0 * i / rot)
    close(f, stretched)
    if rot > 2:
        assert f[0] == 1.0 and abs(f[-1] * 4 / plain[-1] - 1) < 1e-6
    f, a = am.rope_frequencies(rot, base, "parts", 16.0, original=4096)
    keep = np.clip((4096 * plain / (2 * np.pi) - 1) / 31, 0, 1)
    close(f, plain * keep + plain / 16 * (1 - keep))
    assert a == np.float32(1 + 0.1 * np.log(16.0))
    f, a = am.rope_frequencies(rot, base, "parts", 16.0, original=4096, low=2.0, high=8.0)
    keep = np.clip((4096 * plain / (2 * np.pi) - 2) / 6, 0, 1)
    close(f, plain * keep + plain / 16 * (1 - keep))


@pytest.mark.parametrize("args,code", [
    ((3,), -3), ((0,), -3), ((64, 0.0), -9), ((64, float("inf")), -9), ((64, 1e4, "linear", 0.5), -9),
    ((64, 1e4, "base", float("nan")), -9), ((64, 1e4, "parts", 2.0, 0), -2),
    ((64, 1e4, "parts", 2.0, 100, 8.0, 8.0), -9)])
def test_frequency_refusals(am, args, code):
    with pytest.raises(am.AtnError) as e:
        am.rope_frequencies(*args)
    assert e.value.status == code


def arr(shape, dtype="bf16", at=QA, strides=None):
    import hip_rt
    return hip_rt.DeviceArray.wrap(at, shape, dtype, strides=strides)


def test_binding_checks(am):
    K, V = arr((10, 2, 16, 64), at=KA), arr((10, 2, 16, 64), at=VA)
    table, length = arr((3, 4), "i32", TA), arr((3,), "i32", LA)
    c = am.PagedCache(K, V, table, length)
    d = am.Drafts(arr((3, 4, 5, 64)), arr((3, 2, 5, 64), at=KD), arr((3, 2, 5, 64), at=VD))
    r = am.Rotary(arr((32,), "f32", FA), "half")
    assert r.rotary_dim == 64
    out = arr((3, 4, 5, 64), at=OA)
    bad = [
        lambda: am.PagedCache(arr((10, 2, 16)), V, table, length),
        lambda: am.PagedCache(K, arr((10, 2, 16, 32)), table, length),
        lambda: am.PagedCache(K, V, arr((3, 4), "f32"), length),
        lambda: am.PagedCache(K, V, arr((12,), "i32"), length),
        lambda: am.PagedCache(K, V, table, arr((2,), "i32")),
        lambda: am.PagedCache(arr((10, 2, 16, 64), strides=(4096, 2048, 128, 2)), V, table, length),
        lambda: am.Rotary(arr((32,), "f32"), "half", 66),
        lambda: am.Rotary(arr((32,), "bf16")),
        lambda: am.Rotary(arr((4, 8), "f32")),
        lambda: am.SharedPrefix(arr((3,), "i32"), arr((3,), "i32")),
        lambda: am.SharedPrefix(arr((3,), "f32"), arr((2,), "i32")),
        lambda: am.paged_attention_call(c, am.Drafts(arr((2, 4, 5, 64))), out),
        lambda: am.paged_attention_call(c, am.Drafts(arr((3, 3, 5, 64))), arr((3, 3, 5, 64))),
        lambda: am.paged_attention_call(c, am.Drafts(arr((3, 4, 5, 32))), out),
        lambda: am.paged_attention_call(c, d, arr((3, 4, 5, 32))),
        lambda: am.paged_attention_call(c, d, out, lse=arr((3, 4), "f32")),
        lambda: am.paged_append_call(c, d, r, pos=arr((3,), "i32")),
        lambda: am.paged_append_call(c, d, r, q_out=arr((3, 2, 5, 64))),
        lambda: am.paged_append_call(
            c, am.Drafts(arr((3, 4, 5, 64)), arr((3, 4, 5, 64)), arr((3, 4, 5, 64))), r),
        lambda: am.rotary_call(r, [(d.Q, arr((3, 4, 5, 32)))]),
        lambda: am.rotary_call(r, [(d.Q, out), (arr((3, 4, 6, 64)), out)]),
        lambda: am.rotary_call(r, [(d.Q, out)], pos=arr((3, 4), "i32")),
        lambda: am.rotary_call(r, [(d.Q, out)] * 4)]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"case {i} was accepted")
    assert am.paged_attention_workspace_bytes(c, d) >= 40960
    # calls may be made of what a GPU will read later
    assert am.paged_append_call(c, d, r, q_out=d.Q).name == "atn_paged_append_ex"
    assert am.rotary_call(r, [(d.Q, d.Q), (d.K, d.K)], inverse=True).name == "atn_rotary_ex"


def test_division_by_multiplication():
    """The kernels' x / d for x < 2^31: the high word of x times ceil(2^(31 + l) / d), shifted."""
    rng = np.random.default_rng(3)
    ds = list(range(2, 70)) + [int(2 ** rng.uniform(1, 30)) for _ in range(300)] + \
        [2 ** k + e for k in range(2, 30) for e in (-1, 0, 1)]
    for d in ds:
        l = (d - 1).bit_length()
        m = -(-(1 << (31 + l)) // d)
        assert m < 1 << 32
        q = rng.integers(0, (1 << 31) // d, 50)
        x = np.unique(np.concatenate([q * d, q * d + d - 1, [0, (1 << 31) - 1]]))
        for v in x[x < 1 << 31].tolist():
            assert (v * m >> 32) >> (l - 1) == v // d


@pytest.mark.parametrize("B,T", [(1, 1), (2, 1), (32, 1), (2, 2), (3, 5)])
def test_columns_of_one_buffer(am, B, T):
    """Queries, keys and values as columns of a projection's rows, one token a sequence or several."""
    ok = no_device(am)
    if ok == 0:
        pytest.skip("addresses that nothing may dereference")
    row = (4 + 2 + 2) * 64
    s = (T * row, 64, row)
    c = cache(am, batch=B)

    def of(k):  # K's first column
        return drafts(am, tokens=T, Q=QA, K=QA + 2 * k, V=QA + 2 * 6 * 64, q_stride=s, k_stride=s, v_stride=s)

    assert append(am, c, of(4 * 64), rotary(am), q_out=QA, st=s) == ok
    assert append(am, c, of(4 * 64 - 1), rotary(am), q_out=QA, st=s) == -5
    x = [dict(inp=QA, out=QA, in_stride=s, out_stride=s),
         dict(inp=QA + 512, out=QA + 512, in_stride=s, out_stride=s, heads=2)]
    assert rotate(am, x, rotary(am), B=B, T=T) == ok
    x[1].update(inp=QA + 510, out=QA + 510)
    assert rotate(am, x, rotary(am), B=B, T=T) == -5
    # (the last row's columns behind the buffer's rows: the next sequence's queries)
    x[1].update(inp=QA + 2 * (row - 64), out=QA + 2 * (row - 64))
    assert rotate(am, x, rotary(am), B=B, T=T) == (-5 if B * T > 1 else ok)


def test_layouts_of_one_buffer(am):
    """Two tensors in one buffer, in any order of its dimensions: refused where they have an element in
    common, by the sets of their elements."""
    ok = no_device(am)
    if ok == 0:
        pytest.skip("addresses that nothing may dereference")
    rng = np.random.default_rng(11)
    r = rotary(am, rotary_dim=2)
    seen = {-5: 0, ok: 0}
    for _ in range(3000):
        B, T, D = (int(x) for x in rng.choice([1, 2, 3, 4], 3))
        D += D % 2
        heads = [int(x) for x in rng.integers(1, 4, 2)]
        sizes = dict(b=B + int(rng.integers(0, 2)), h=sum(heads) + int(rng.integers(0, 2)), t=T)
        at, s = D + int(rng.integers(0, 3)), {}
        for d in rng.permutation(list("bht")):
            s[d] = at
            at *= sizes[d]
        st = (s["b"], s["h"], s["t"])
        first = [0, heads[0] * s["h"]]
        if rng.random() < 0.5:
            first[1] = int(rng.integers(0, at))
        first = first if rng.random() < 0.5 else first[::-1]
        e = [set((f + s["b"] * np.arange(B)[:, None, None, None] + s["h"] * np.arange(h)[:, None, None] +
                  s["t"] * np.arange(T)[:, None] + np.arange(D)).ravel().tolist())
             for f, h in zip(first, heads)]
        x = [dict(inp=QA + 2 * f, out=QA + 2 * f, in_stride=st, out_stride=st, heads=h)
             for f, h in zip(first, heads)]
        want = -5 if e[0] & e[1] else ok
        assert rotate(am, x, r, B=B, T=T, D=D) == want, (B, T, D, heads, st, first)
        seen[want] += 1
    assert min(seen.values()) > 500


@pytest.mark.parametrize("c,code", [
    (dict(V=KA + 64), -5), (dict(V=KA + 2), -5), (dict(V=KA - 2 * 9 * 2048 - 2), -5),
    (dict(V=KA + 2 * 10 * 2048 - 2), -5), (dict(V=KA + 2 * 10 * 2048), 0),
    # V behind K in every page, in every page's every row, and one element too near
    (dict(V=KA + 4096, k_stride=(4096, 1024, 64), v_stride=(4096, 1024, 64)), 0),
    (dict(V=KA + 4094, k_stride=(4096, 1024, 64), v_stride=(4096, 1024, 64)), -5),
    (dict(V=KA + 4096, k_stride=(4096, 1024, 64), v_stride=(4096, 64, 128)), 0),
    (dict(V=KA + 128, k_stride=(4096, 2048, 128), v_stride=(4096, 2048, 128)), 0),
    (dict(V=KA + 126, k_stride=(4096, 2048, 128), v_stride=(4096, 2048, 128)), -5),
    (dict(V=KA + 128, k_stride=(4096, 2048, 128), v_stride=(4096, 2048, 130)), -5)])
def test_append_to_overlapping_pools(am, c, code):
    ok = no_device(am)
    if ok == 0:
        pytest.skip("addresses that nothing may dereference")
    assert append(am, cache(am, **c), drafts(am), rotary(am)) == (code or ok)


def need(am, c, d, p=None, n=0):
    return am.lib().atn_paged_attention_workspace_bytes(ref(c), ref(d), ref(p), n)


WS = 0x7E0000000000


def test_workspace_of_a_larger_bound(am):
    """A workspace asked for with one bound of the lengths serves every smaller one, where dims are
    shared by several workgroups (each share has scores of its own) too."""
    if no_device(am) == 0:
        pytest.skip("addresses that nothing may dereference")
    import random
    rng = random.Random(5)
    cases = [dict(D=8192, dt=0, B=1, G=1, rep=1, T=1, page=16, slots=1100, bounds=[16400, 4000]),
             dict(D=2048, dt=0, B=1, G=1, rep=1, T=1, page=16, slots=1300, bounds=[20000, 16000])]
    for _ in range(600):
        D, page, slots = rng.choice([80, 128, 512, 2048, 8192]), rng.choice([16, 20]), \
            int(2 ** rng.uniform(2, 10))
        cases.append(dict(D=D, dt=rng.choice([0, 1]), B=int(2 ** rng.uniform(0, 5)), G=rng.choice([1, 2, 8]),
                          rep=rng.choice([1, 4, 8]), T=int(2 ** rng.uniform(0, 9)), page=page, slots=slots,
                          bounds=sorted((rng.randint(1, page * slots) for _ in range(4)), reverse=True)))
    for x in cases:
        c = cache(am, dtype=x["dt"], batch=x["B"], kv_heads=x["G"], pages=1 << 14, page_rows=x["page"],
                  table_pages=x["slots"], head_d=x["D"])
        d = drafts(am, heads=x["G"] * x["rep"], tokens=x["T"])
        for p in (None, prefix(am, groups=(x["B"] + 1) // 2)):
            for i, most in enumerate(x["bounds"]):
                n = need(am, c, d, p, most)
                assert n > 0
                for less in x["bounds"][i:]:
                    assert attend(am, c, d, p, max_len=less, ws=WS, wsb=n) == -6, (x, most, less)


def test_prefixes_that_no_workspace_holds(am):
    """A prefix saves reads and promises another order of sums, no more: where its parts do not fit the
    library's workspace, or no group could save what they cost, the call runs as without it."""
    ok = no_device(am)
    if ok == 0:
        pytest.skip("addresses that nothing may dereference")
    for dtype, B, H, G, T, D, page, slots, groups in [
            (1, 8, 32, 1, 4096, 128, 16, 512, 1), (1, 8, 32, 1, 4096, 128, 16, 4096, 2),
            (1, 16, 64, 8, 8192, 128, 16, 1024, 4), (1, 58, 8, 1, 431, 512, 16, 32, 3),
            (0, 8, 32, 1, 4096, 80, 20, 400, 3), (1, 40, 16, 1, 2048, 256, 16, 300, 20),
            (0, 100, 8, 1, 256, 2048, 20, 8, 70)]:
        c = cache(am, dtype=dtype, batch=B, kv_heads=G, pages=1 << 14, page_rows=page, table_pages=slots,
                  head_d=D)
        d, p = drafts(am, heads=H, tokens=T), prefix(am, groups=groups)
        assert attend(am, c, d) == ok
        assert attend(am, c, d, p) == ok
        n = need(am, c, d, p)
        assert need(am, c, d) <= n <= (1 << 30) + 40960
        assert attend(am, c, d, p, ws=WS, wsb=n) == ok
        # no group of so short rows beside so many queries is read once: no room for one is needed
        least = need(am, c, d)
        assert attend(am, c, d, p, max_len=64, ws=WS, wsb=least) == ok
        # (a larger one than the library's holds them)
        assert attend(am, c, d, p, ws=WS, wsb=1 << 40) == ok


def test_prefixes_where_they_run_without(am):
    """No call with a prefix is refused that runs without it, for want of room in the library's workspace or in
    one that was asked for."""
    if no_device(am) == 0:
        pytest.skip("addresses that nothing may dereference")
    import random
    rng = random.Random(8)
    for _ in range(1500):
        D, page = rng.choice([64, 80, 128, 192, 512, 2048]), rng.choice([16, 20])
        B, rep, T = int(2 ** rng.uniform(1, 6)), rng.choice([1, 4, 8, 32]), int(2 ** rng.uniform(0, 13))
        c = cache(am, dtype=rng.choice([0, 1]), batch=B, kv_heads=rng.choice([1, 2, 8]), pages=1 << 14,
                  page_rows=page, table_pages=int(2 ** rng.uniform(1, 12)), head_d=D)
        d, p = drafts(am, heads=c.kv_heads * rep, tokens=T), prefix(am, groups=rng.randint(1, B))
        plain = attend(am, c, d)
        if plain != -6:
            continue
        assert attend(am, c, d, p) == -6
        n = need(am, c, d, p)
        assert attend(am, c, d, p, ws=WS, wsb=n) == -6
        # ... with any smaller bound of the lengths
        for _ in range(3):
            assert attend(am, c, d, p, max_len=rng.randint(1, page * c.table_pages), ws=WS, wsb=n) == -6


@pytest.mark.parametrize("dtype,B,H,G,T,D,rows", [
    (1, 4, 32, 8, 2048, 512, 8192), (1, 64, 16, 1, 512, 1024, 8192), (0, 16, 8, 8, 4096, 2048, 8192),
    (0, 1000, 4, 1, 300, 512, 4096), (1, 7, 32, 8, 2048, 512, 24576)])
def test_prompts_of_wide_heads(am, dtype, B, H, G, T, D, rows):
    """head_d > 256, scores of all sequences past the library's workspace: sequences in turn."""
    ok = no_device(am)
    if ok == 0:
        pytest.skip("addresses that nothing may dereference")
    c = cache(am, dtype=dtype, batch=B, kv_heads=G, pages=1 << 16, page_rows=16,
              table_pages=rows // 16, head_d=D)
    d = drafts(am, heads=H, tokens=T)
    assert 40960 < need(am, c, d) <= (1 << 30) + 40960
    assert attend(am, c, d) == ok
    assert attend(am, c, d, prefix(am, groups=2)) == ok
    # one sequence's scores of one kv head have to fit
    one = 4 * (H // G) * T * rows
    assert attend(am, c, d, ws=WS, wsb=one + (one >> 4)) == ok
    assert attend(am, c, d, ws=WS, wsb=one // 2) == -8


def test_rotary_call_of_no_tensors(am):
    with pytest.raises(ValueError):
        am.rotary_call(am.Rotary(arr((32,), "f32", FA)), [])


@pytest.mark.parametrize("D,B,rep,T,slots,groups,bounds", [
    (8, 244, 1, 76, 71, 67, [1136, 511, 300, 20]), (8, 504, 8, 11, 202, 186, [3232, 2759, 511, 500]),
    (64, 476, 1, 69, 164, 100, [2624, 2500, 511, 100])])
def test_workspace_of_a_larger_bound_and_smaller_tiles(am, D, B, rep, T, slots, groups, bounds):
    """Prefixes whose tiles, and so the parts, grow where the bound of the lengths shrinks."""
    if no_device(am) == 0:
        pytest.skip("addresses that nothing may dereference")
    c = cache(am, batch=B, kv_heads=1, pages=1 << 14, table_pages=slots, head_d=D)
    d, p = drafts(am, heads=rep, tokens=T), prefix(am, groups=groups)
    for i, most in enumerate(bounds):
        n = need(am, c, d, p, most)
        for less in bounds[i:]:
            assert attend(am, c, d, p, max_len=less, ws=WS, wsb=n) == -6
