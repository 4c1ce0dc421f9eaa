"""Decoding over a cache, without a GPU: every argument error is reported with its status before
any HIP call, workspace queries, the binding's checks, and tree masks."""
import ctypes

import numpy as np
import pytest

# device addresses that nothing dereferences
KA, VA, QA, KD, VD, OA, LA, NA, WA, PA, SA, XA = (0x7F0000000000 + i * 0x1000000000
                                                  for i in range(12))


def cache(am, **kw):
    f = dict(K=KA, V=VA, len=LA, seen=SA, weight=WA, pos=PA, dtype=1, batch=2, kv_heads=2,
             capacity=100, head_d=64)
    f.update(kw)
    c = am._KvCacheDesc()
    for k, v in f.items():
        setattr(c, k, (ctypes.c_int64 * 3)(*v) if k.endswith("stride") else v)
    return c


def drafts(am, **kw):
    f = dict(Q=QA, K=KD, V=VD, heads=4, tokens=5)
    f.update(kw)
    d = am._DraftsDesc()
    for k, v in f.items():
        setattr(d, k, (ctypes.c_int64 * 3)(*v) if k.endswith("stride") else v)
    return d


def ref(x):
    return None if x is None else ctypes.byref(x)




def calls(am):
    L = am.lib()

    def attend(c, d, out=OA, strides=None, lse=NA, scale=0.0, max_len=0, ws=None, wsb=0):
        s = (ctypes.c_int64 * 3)(*strides) if strides else None
        return L.atn_tree_attention_ex(ref(c), ref(d), out, ctypes.cast(s, ctypes.c_void_p) if s
                                       else None, lse, scale, max_len, ws, wsb, None)

    def commit(c, d, path=XA, accepted=XA, n=4):
        return L.atn_cache_commit_ex(ref(c), ref(d), path, accepted, n, None)

    def weigh(c, d, lse=NA, path=XA, accepted=XA, n=4, win=None, scale=0.0, max_len=0):
        return L.atn_cache_weigh_ex(ref(c), ref(d), lse, path, accepted, n, win, scale, max_len, None)

    def evict(c, d=None, budget=50, recent=5, ws=None, wsb=0):
        return L.atn_cache_evict_ex(ref(c), budget, recent, ws, wsb, None)

    def advance(c, d, path=XA, accepted=XA, n=4, limit=0):
        return L.atn_cache_advance_ex(ref(c), ref(d), path, accepted, n, limit, None)

    return dict(attend=attend, commit=commit, weigh=weigh, evict=evict, advance=advance)


ALL = ["attend", "commit", "weigh", "evict", "advance"]


@pytest.mark.parametrize("op", ALL)
@pytest.mark.parametrize("kw,code", [
    (dict(dtype=2), -9), (dict(dtype=-1), -9), (dict(K=None), -1), (dict(V=None), -1),
    (dict(len=None), -1), (dict(batch=0), -2), (dict(kv_heads=0), -2), (dict(capacity=0), -2),
    (dict(head_d=0), -2), (dict(capacity=-4), -2), (dict(head_d=8193), -9),
    (dict(batch=65536, kv_heads=2), -4), (dict(batch=1 << 30, kv_heads=1 << 30), -4),
    (dict(K=KA + 1), -10), (dict(V=VA + 1), -10), (dict(len=LA + 2), -10), (dict(weight=WA + 1), -10),
    (dict(pos=PA + 2), -10), (dict(seen=SA + 3), -10),
    (dict(k_stride=(-1, 6400, 64)), -9), (dict(v_stride=(12800, 6400, 63)), -9),   # rows overlap
    (dict(k_stride=(12800, 64, 64)), -9), (dict(k_stride=(0, 6400, 64)), -9),      # heads, batches
    (dict(k_stride=(12800, 6400, 0)), -9), (dict(k_stride=(1 << 62, 6400, 64)), -4),
    (dict(v_stride=(1 << 61, 1 << 61, 64)), -4)])
def test_cache_refusals(am, op, kw, code):
    assert calls(am)[op](cache(am, **kw), drafts(am)) == code


@pytest.mark.parametrize("op", ["attend", "commit", "weigh", "advance"])
@pytest.mark.parametrize("kw,code", [
    (dict(heads=0), -2), (dict(tokens=0), -2), (dict(heads=3), -9), (dict(heads=1), -9),
    (dict(tokens=257), -9), (dict(K=None), -1), (dict(V=None), -1), (dict(count=LA + 1), -10),
    (dict(mask=LA + 2), -10), (dict(K=KD + 1), -10), (dict(k_stride=(640, -320, 64)), -9),
    (dict(v_stride=(1 << 62, 320, 64)), -4)])
def test_drafts_refusals(am, op, kw, code):
    assert calls(am)[op](cache(am), drafts(am, **kw)) == code


def test_null_descriptors(am):
    f = calls(am)
    for op in ALL:
        assert f[op](None, drafts(am)) == -1
    for op in ("attend", "commit", "weigh"):
        assert f[op](cache(am), None) == -1
    assert f["advance"](cache(am), None) == -9  # neither rows nor a limit


@pytest.mark.parametrize("kw,dkw,code", [
    (dict(out=None), {}, -1), ({}, dict(Q=None), -1), (dict(out=OA + 1), {}, -10),
    (dict(lse=NA + 2), {}, -10), ({}, dict(Q=QA + 1), -10), (dict(scale=float("nan")), {}, -9),
    (dict(scale=float("inf")), {}, -9), (dict(scale=3e38), {}, -9), (dict(max_len=-1), {}, -2),
    (dict(out=QA), {}, -5), (dict(out=KA + 64), {}, -5), (dict(out=VD), {}, -5),
    (dict(out=VA - 2), {}, -5), (dict(lse=QA), {}, -5), (dict(lse=OA + 256), {}, -5),
    (dict(strides=(1280, 320, 0)), {}, -9), (dict(strides=(0, 320, 64)), {}, -9),
    (dict(strides=(1280, 320, 63)), {}, -9), (dict(strides=(-1, 320, 64)), {}, -9),
    (dict(ws=XA, wsb=100), {}, -8)])
def test_attention_refusals(am, kw, dkw, code):
    assert calls(am)["attend"](cache(am), drafts(am, **dkw), **kw) == code


@pytest.mark.parametrize("op", ["commit", "weigh", "advance"])
@pytest.mark.parametrize("kw,code", [(dict(n=0), -2), (dict(n=257), -9), (dict(path=XA + 1), -10),
                                     (dict(accepted=XA + 2), -10)])
def test_path_refusals(am, op, kw, code):
    assert calls(am)[op](cache(am), drafts(am), **kw) == code


def test_commit_refusals(am):
    f = calls(am)["commit"]
    assert f(cache(am), drafts(am, K=None, V=None)) == -1
    assert f(cache(am, seen=None), drafts(am)) == -1       # positions need the tokens seen
    assert f(cache(am, V=KA), drafts(am)) == -5            # one tensor for both
    assert f(cache(am), drafts(am, K=KA + 1024)) == -5
    assert f(cache(am), drafts(am, V=KA + 1024)) == -5


def test_weigh_refusals(am):
    f = calls(am)["weigh"]
    assert f(cache(am), drafts(am), lse=None) == -1
    assert f(cache(am, weight=None), drafts(am)) == -1
    assert f(cache(am), drafts(am, Q=None)) == -1
    assert f(cache(am), drafts(am), lse=NA + 1) == -10
    assert f(cache(am), drafts(am), win=XA + 1) == -10
    assert f(cache(am), drafts(am), win=WA + 4) == -5      # neither in place nor apart
    assert f(cache(am, weight=KA + 64), drafts(am)) == -5
    assert f(cache(am), drafts(am), lse=WA + 400) == -5
    assert f(cache(am), drafts(am), scale=float("nan")) == -9
    assert f(cache(am), drafts(am), max_len=-7) == -2


def test_evict_refusals(am):
    f = calls(am)["evict"]
    for missing in ("weight", "pos", "seen"):
        assert f(cache(am, **{missing: None})) == -1
    assert f(cache(am), budget=0) == -2 and f(cache(am), budget=-3) == -2
    assert f(cache(am), recent=-1) == -9 and f(cache(am), recent=51) == -9
    assert f(cache(am, V=KA)) == -5
    assert f(cache(am, weight=KA + 4)) == -5
    assert f(cache(am, pos=WA + 4)) == -5


def test_advance_refusals(am):
    f = calls(am)["advance"]
    assert f(cache(am), drafts(am), limit=-1) == -2
    assert f(cache(am), None, limit=0) == -9


def test_valid_calls_reach_the_device(am):
    if am.device_count() > 0:
        pytest.skip("a device is present")
    f = calls(am)
    ok = am.ATN_ERR_NO_DEVICE
    c, d = cache(am), drafts(am)
    assert f["attend"](c, d) == ok and f["attend"](c, d, lse=None) == ok
    assert f["attend"](c, drafts(am, K=None, V=None)) == ok
    assert f["attend"](c, drafts(am, q_stride=(1280, 64, 256), k_stride=(0, 0, 64)),
                       strides=(1280, 64, 256)) == ok      # tokens outside heads; shared drafts
    assert f["attend"](cache(am, V=KA), d) == ok           # one tensor for keys and values
    assert f["attend"](cache(am, k_stride=(12800, 64, 128), v_stride=(25600, 64, 256)), d) == ok
    assert f["commit"](c, d) == ok and f["commit"](c, d, path=None, accepted=None) == ok
    assert f["commit"](cache(am, seen=None, pos=None, weight=None), d) == ok
    assert f["weigh"](c, d) == ok and f["weigh"](c, d, win=WA) == ok
    assert f["weigh"](c, drafts(am, K=None, V=None), win=XA) == ok
    assert f["evict"](c) == ok and f["evict"](c, budget=500, recent=0) == ok
    assert f["advance"](c, d) == ok and f["advance"](c, None, limit=3) == ok


def test_workspace_queries(am):
    L = am.lib()
    c, d = cache(am), drafts(am)
    w = L.atn_tree_attention_workspace_bytes
    assert w(ref(c), ref(d), 0) >= 40960
    assert w(ref(cache(am, head_d=0)), ref(d), 0) == 0 and w(ref(c), None, 0) == 0
    assert w(ref(c), ref(d), -1) == 0
    e = L.atn_cache_evict_workspace_bytes
    assert e(ref(c), 50) >= 40960 + 2 * 2 * (1 + 2 * 50) * 4
    assert e(ref(c), 0) == 0 and e(None, 5) == 0


def test_tree_mask(am):
    m = am.tree_mask([[-1, 0, 0, 2, -1], [-1, 0, 1, 2, 3]])
    assert m.shape == (2, 5, 1) and m.dtype == np.int32
    assert m[0, :, 0].tolist() == [1, 3, 5, 13, 16] and m[1, :, 0].tolist() == [1, 3, 7, 15, 31]
    m = am.tree_mask([list(range(-1, 69))])
    assert m.shape == (1, 70, 3)
    assert m[0, 69].view(np.uint32).tolist() == [0xffffffff, 0xffffffff, 0x3f]
    with pytest.raises(ValueError):
        am.tree_mask([[-1, 1]])
    with pytest.raises(ValueError):
        am.tree_mask([[-2, 0]])




def test_binding_checks(am):
    """Shapes, types and strides that do not fit are ValueErrors before any call."""
    import hip_rt

    def arr(shape, dtype="bf16", strides=None, ptr=KA):
        return hip_rt.DeviceArray.wrap(ptr, shape, dtype, strides)

    K, V, n = arr((2, 2, 100, 64)), arr((2, 2, 100, 64), ptr=VA), arr((2,), "i32")
    c = am.KvCache(K, V, n, seen=n, weight=arr((2, 2, 100), "f32"), pos=arr((2, 2, 100), "i32"))
    for bad in (lambda: am.KvCache(K, arr((2, 2, 99, 64)), n), lambda: am.KvCache(K, V, arr((3,), "i32")),
                lambda: am.KvCache(K, V, arr((2,), "f32")), lambda: am.KvCache(arr((2, 100, 64)), V, n),
                lambda: am.KvCache(K, V, n, weight=arr((2, 2, 99), "f32")),
                lambda: am.KvCache(arr((2, 2, 100, 64), strides=(25600, 12800, 128, 2)), V, n)):
        with pytest.raises(ValueError):
            bad()
    Q, kd = arr((2, 4, 5, 64)), arr((2, 2, 5, 64))
    d = am.Drafts(Q, kd, kd)
    for bad in (lambda: am.Drafts(Q, kd, None), lambda: am.Drafts(Q, kd, arr((2, 2, 4, 64))),
                lambda: am.Drafts(Q, mask=arr((2, 5, 2), "i32")), lambda: am.Drafts(Q, count=arr((1,), "i32")),
                lambda: am.tree_attention_call(c, am.Drafts(arr((2, 3, 5, 64)))),
                lambda: am.tree_attention_call(c, am.Drafts(arr((2, 4, 5, 32)))),
                lambda: am.tree_attention_call(c, am.Drafts(arr((2, 4, 5, 64), "f32"))),
                lambda: am.tree_attention_call(c, am.Drafts(Q, arr((2, 4, 5, 64)), arr((2, 4, 5, 64)))),
                lambda: am.tree_attention_call(c, d, arr((2, 4, 5, 63))),
                lambda: am.tree_attention_call(c, d, Q, lse=arr((2, 4, 4), "f32")),
                lambda: am.cache_commit_call(c, d, path=arr((3, 4), "i32")),
                lambda: am.cache_commit_call(c, d, accepted=arr((3,), "i32")),
                lambda: am.cache_weigh_call(c, d, arr((2, 4, 5), "i32")),
                lambda: am.attention_ex(arr((2, 2, 100, 64), strides=(1, 2, 3, 1)), K, V, V)):
        with pytest.raises(ValueError):
            bad()


def test_host_arrays_of_int32(am):
    import hip_rt
    assert hip_rt.contiguous_strides((2, 3, 4)) == (12, 4, 1)
    a = hip_rt.DeviceArray.wrap(KA, (2, 3), "i32", (3, 1))
    assert a.strides is None and a.nbytes == 24
    assert hip_rt.DeviceArray.wrap(KA, (2, 3), "i32", (4, 1)).strides == (4, 1)


def test_sizes_past_the_kernels_numbers(am):
    """Rows more than 128 MiB apart, more than 2^30 rows, more blocks than an int counts, and
    scales that fp32 does not hold as normal numbers."""
    f = calls(am)
    ld = (1 << 26) + 1  # bf16 elements: 128 MiB and one more
    far = dict(batch=1, kv_heads=1, capacity=4)
    for op in ALL:
        assert f[op](cache(am, k_stride=(0, 0, ld), **far), drafts(am)) == -4
        assert f[op](cache(am, v_stride=(0, 0, ld), **far), drafts(am)) == -4
        assert f[op](cache(am, batch=1, kv_heads=1, capacity=(1 << 30) + 1, head_d=1), drafts(am)) == -4
    assert f["attend"](cache(am), drafts(am, k_stride=(0, 0, ld))) == -4
    assert f["attend"](cache(am), drafts(am, v_stride=(0, 0, ld))) == -4
    wide = drafts(am, heads=1 << 17, tokens=1)
    assert f["weigh"](cache(am, batch=1, kv_heads=1, head_d=1), wide, n=128) == -4
    small = [(1 << 40) * i for i in range(20, 32)]
    c = cache(am, K=small[0], V=small[0], len=small[6], seen=None, weight=None, pos=None, batch=100,
              kv_heads=1, capacity=1 << 30, head_d=1)
    d = drafts(am, Q=small[8], K=small[9], V=small[10], heads=1, tokens=1)
    assert f["attend"](c, d, out=small[11], lse=None) == -4
    for scale in (1e-39, -1e-40, 1e-45):
        assert f["attend"](cache(am), drafts(am), scale=scale) == -9
        assert f["weigh"](cache(am), drafts(am), scale=scale) == -9


def test_grids_past_the_hardware(am):
    """More workgroups than a grid's dimension holds threads for."""
    c = cache(am, batch=65535, kv_heads=1, capacity=1, head_d=1)
    d = drafts(am, heads=512, tokens=32)
    assert calls(am)["attend"](c, d, lse=None) == -4


def test_strides_of_single_rows(am):
    """A dimension of one element may have any stride, 0 among them."""
    import hip_rt
    one = hip_rt.DeviceArray.wrap(KA, (1, 1, 1, 64), "bf16", (0, 0, 0, 1))
    am.KvCache(one, one, hip_rt.DeviceArray.wrap(LA, (1,), "i32"))
    with pytest.raises(ValueError):
        am.Drafts(hip_rt.DeviceArray.wrap(QA, (1, 2, 1, 64), "bf16", (0, 0, 0, 1)))


def test_commit_refuses_tables_inside_the_tensors(am):
    f = calls(am)["commit"]
    assert f(cache(am, weight=KA + 64), drafts(am)) == -5
    assert f(cache(am, pos=VA + 64), drafts(am)) == -5
    assert f(cache(am, weight=KD), drafts(am)) == -5
    assert f(cache(am, pos=WA + 4), drafts(am)) == -5
