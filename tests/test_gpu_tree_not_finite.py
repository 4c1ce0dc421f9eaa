"""Attention of drafted tokens over infinities and NaN in V: those of a key that a token attends
reach its output as they are, in their dims, however small the key's weight and wherever it lies;
a token without a score above -infinity gets zeros."""
import numpy as np
import pytest

import cache_helpers as C
from test_gpu_tree_attention import Problem

pytestmark = pytest.mark.gpu

FAR = 400.0  # exp(-400) is 0 in fp32, and a bf16 number

# of every kernel: waves alone with whole pairs and with ranges, shared blocks of 128 and 256
# rows, scores and values apart with tiles of 16 and 32 rows
SHAPES = [("bf16", 48, 2, 3), ("f32", 48, 2, 3), ("bf16", 128, 2, 3), ("f32", 128, 2, 20),
          ("bf16", 100, 4, 20), ("bf16", 128, 4, 50), ("bf16", 200, 2, 20), ("f32", 200, 2, 3),
          ("bf16", 300, 2, 3), ("f32", 520, 4, 10), ("bf16", 4, 2, 3)]


def place(p, q, k, kd, v, vd):
    """The problem's tensors set to these."""
    for t, x in ((p.Q, q), (p.K, k), (p.Kd, kd), (p.V, v), (p.Vd, vd)):
        t.host = C.rounded(x, p.dtype)
        t.base.upload(t._flat(t.host))


def tensors(p):
    return [t.host.copy() for t in (p.Q, p.K, p.Kd, p.V, p.Vd)]


def check(p):
    """Against the definition: the sum of what is not finite where a token attends any in that dim,
    elsewhere the finite values' result."""
    v, vd = p.V.host, p.Vd.host
    B, H, T, D = p.Q.host.shape
    rep = H // v.shape[1]
    odd = np.zeros((B, H, T, D))
    with np.errstate(invalid="ignore"):
        only, only_d = (np.where(np.isfinite(x), 0.0, x) for x in (v, vd))
        for b, (L, n) in enumerate(zip(p.lens, p.counts)):
            see = C.visible(T, n, p.words, b)
            for h in range(H):
                g = h // rep
                rows = only[b, g, :L].sum(0)
                for t in range(n):
                    odd[b, h, t] = rows + only_d[b, g][see[t]].sum(0)
    p.V.host, p.Vd.host = np.where(np.isfinite(v), v, 0), np.where(np.isfinite(vd), vd, 0)
    want, want_lse, _ = p.want(scale=1.0)
    out, lse = p.out.numpy(), p.lse.numpy()
    # (the tolerances of finite scores: one of -infinity is exact)
    p.K.host, p.Kd.host = (np.where(np.isneginf(x.host), -FAR, x.host) for x in (p.K, p.Kd))
    tol, tol_lse = C.attend_tol(p.dtype, D, want, p.want(scale=1.0)[2])
    for b, n in enumerate(p.counts):
        o, w, s = out[b, :, :n], want[b, :, :n], odd[b, :, :n]
        nothing = np.isneginf(want_lse[b, :, :n])
        assert np.array_equal(nothing, np.isneginf(lse[b, :, :n]))
        assert (o[nothing] == 0).all()
        f = np.isfinite(s) & ~nothing[..., None]
        assert (np.abs(o - w)[f] <= tol[b, :, :n][f]).all()
        x = ~np.isfinite(s) & ~nothing[..., None]
        assert np.array_equal(o[x], s[x].astype(np.float32), equal_nan=True), \
            f"{(o[x] != s[x]).sum()} of {x.sum()}: {o[x][:6]} for {s[x][:6]}"
        ok = ~nothing
        e = np.abs(lse[b, :, :n][ok] - want_lse[b, :, :n][ok])
        assert (e <= tol_lse[b, :, :n][ok] + 4 * C.U32 * np.abs(want_lse[b, :, :n][ok])).all()


def start(p):
    """Queries with 1 in dim 0, keys with 0: a key's dim 0 is added to its scores."""
    q, k, kd, v, vd = tensors(p)
    q[..., 0], k[..., 0], kd[..., 0] = 1.0, 0.0, 0.0
    return q, k, kd, v, vd


def mark(v, vd, b, L, D):
    """What is not finite, in dims of its own: the cache's first, middle and last row, opposite
    infinities in two of them, and drafts that all or only the last tokens attend."""
    put = [(v, 0, np.inf), (v, L // 2, -np.inf), (v, L - 1, np.inf), (vd, 0, -np.inf),
           (vd, vd.shape[2] - 1, np.nan)]
    for i, (x, row, y) in enumerate(put):
        x[b, :, row, (3 + 7 * i) % D] = y
    if D > 4:
        v[b, :, 0, D - 1], v[b, :, L - 1, D - 1] = np.inf, -np.inf
        v[b, :, L // 2, D - 2] = np.nan


@pytest.mark.parametrize("dtype,D,Hq,T", SHAPES)
@pytest.mark.parametrize("L", [41, 64, 700, 3001])
@pytest.mark.parametrize("peak", ["first", "last", "draft", "others"])
def test_values_of_vanishing_weight(am, dev, dtype, D, Hq, T, L, peak):
    """One key's score is 400 above the others', or those of the marked keys 400 below: their
    weights are 0 in fp32, also where the running maximum rises only after them."""
    print(f"[case] vanishing {dtype} {D} {Hq} {T} {L} {peak}", flush=True)
    p = Problem(am, dtype, 2, Hq, 1, T, D, L + 3, [L, 37], mask="chain", sigma=0.3, seed=L + D,
                fill=np.nan)
    q, k, kd, v, vd = start(p)
    for b, n in enumerate(p.lens):
        mark(v, vd, b, n, D)
        if peak == "first":
            k[b, :, 1, 0] = FAR
        elif peak == "last":
            k[b, :, n - 2, 0] = FAR
        elif peak == "draft":
            kd[b, :, 0, 0] = FAR
        else:
            k[b, :, [0, n // 2, n - 1], 0] = -FAR
            kd[b, :, [0, T - 1], 0] = -FAR
    place(p, q, k, kd, v, vd)
    p.run(scale=1.0)
    check(p)


@pytest.mark.parametrize("dtype,D,Hq,T", SHAPES)
@pytest.mark.parametrize("L", [41, 64, 700, 3001])
@pytest.mark.parametrize("one", [False, True])
def test_values_without_a_score(am, dev, dtype, D, Hq, T, L, one):
    """Scores of -infinity: alone they are nothing to attend, whatever V holds; beside one that is
    finite (one) their values are attended with the others."""
    print(f"[case] no score {dtype} {D} {Hq} {T} {L} {one}", flush=True)
    p = Problem(am, dtype, 2, Hq, 1, T, D, L + 3, [L, 37], mask="chain", sigma=0.3, seed=L + D,
                fill=np.nan)
    q, k, kd, v, vd = start(p)
    for b, n in enumerate(p.lens):
        mark(v, vd, b, n, D)
        k[b, :, :n, 0] = -np.inf
        kd[b, :, :, 0] = -np.inf
        if one:
            k[b, :, n // 3, 0] = 1.0
    place(p, q, k, kd, v, vd)
    p.run(scale=1.0)
    check(p)


@pytest.mark.parametrize("dtype,D,Hq,T", SHAPES)
def test_scores_that_are_no_numbers_stay_so(am, dev, dtype, D, Hq, T):
    """A token with a NaN score has no finite output in any dim, infinities in V or not; the
    tokens of the other kv head are as without it."""
    print(f"[case] NaN score {dtype} {D} {Hq} {T}", flush=True)
    p = Problem(am, dtype, 1, 2 * Hq, 2, T, D, 90, [77], sigma=0.3, seed=D)
    q, k, kd, v, vd = start(p)
    k[0, 0, 50, 0] = np.nan
    v[0, 0, 3, D - 1] = v[0, 0, 76, D // 2] = np.inf
    place(p, q, k, kd, v, vd)
    p.run(scale=1.0)
    out = p.out.numpy()
    assert not np.isfinite(out[0, :Hq]).any() and np.isnan(out[0, :Hq, :, 0]).all()
    want, want_lse, info = p.want(scale=1.0)
    C.attend_close(dtype, D, *[x[:, Hq:] for x in (out, p.lse.numpy(), want, want_lse)],
                   {n: x[:, Hq:] for n, x in info.items()}, [T])
