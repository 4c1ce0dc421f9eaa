"""The accuracy check of the decoding operators, without a GPU: fp32 arithmetic passes it, and
operands or weights rounded to bf16 anywhere fail it at every head size from 64 up."""
import numpy as np
import pytest

import cache_accuracy as A
import cache_helpers as C

DIMS = [64, 65, 80, 96, 100, 128, 130, 160, 192, 200, 256, 257, 264, 384, 500, 512, 1000, 1024, 2048,
        4100, 8192]
B, H, G, T, LENS = 2, 4, 2, 3, [77, 33]


def inputs(D):
    rng = np.random.default_rng(D)
    return [rng.standard_normal((B, h, n, D)).astype(np.float32) * np.float32(s)
            for h, n, s in ((H, T, 1.5), (G, 77, 1), (G, 77, 1), (G, T, 1), (G, T, 1))]


def attend(Q, K, V, Kd, Vd, t=np.float32, round_weights=False):
    """A chain of drafts over the cache in arithmetic of type t."""
    D = Q.shape[3]
    out, lse = np.zeros(Q.shape), np.zeros(Q.shape[:3])
    for b, L in enumerate(LENS):
        for h in range(H):
            g = h // (H // G)
            for i in range(T):
                k = np.concatenate([K[b, g, :L], Kd[b, g, :i + 1]]).astype(t)
                v = np.concatenate([V[b, g, :L], Vd[b, g, :i + 1]]).astype(t)
                s = (k @ Q[b, h, i].astype(t)) * t(1 / np.sqrt(D))
                m = s.max()
                e = np.exp(s - m)
                lse[b, h, i] = m + np.log(e.sum())
                if round_weights:
                    e = C.rounded(e, "bf16").astype(t)
                out[b, h, i] = e @ v / e.sum()
    return out, lse


def bf16(x):
    return C.rounded(x, "bf16")


@pytest.mark.parametrize("D", DIMS)
def test_the_check_tells_fp32_from_bf16(D):
    Q, K, V, Kd, Vd = inputs(D)
    want, want_lse, info = C.attend64(Q, K, V, Kd, Vd, LENS, [T] * B)
    rows, keys = A.score_rms(Q, K, Kd, LENS), info["keys"].max()
    A.attend_accurate("f32", *attend(Q, K, V, Kd, Vd), want, want_lse, rows, keys)
    # an lse of rounded scores, an output of rounded operands or weights
    scores = attend(bf16(Q), bf16(K), V, bf16(Kd), Vd, np.float64)
    assert A.out_error(scores[0], want) > 10 * A.out_tol("f32", rows, keys)
    assert A.rms(scores[1] - want_lse) > 10 * A.lse_tol(rows, keys, want_lse)
    for bad in (attend(Q, K, bf16(V), Kd, bf16(Vd), np.float64),
                attend(Q, K, V, Kd, Vd, np.float64, round_weights=True)):
        assert A.out_error(bad[0], want) > 10 * A.out_tol("f32", rows, keys)
        with pytest.raises(AssertionError):
            A.attend_accurate("f32", *bad, want, want_lse, rows, keys)
    # outputs of bf16 inputs: rounded weights and output pass, values rounded twice over do not
    got = attend(*map(bf16, (Q, K, V, Kd, Vd)), np.float64, round_weights=True)
    ref = C.attend64(*map(bf16, (Q, K, V, Kd, Vd)), LENS, [T] * B)
    A.attend_accurate("bf16", bf16(got[0]), got[1], ref[0], ref[1], rows, keys)
    with pytest.raises(AssertionError):
        A.attend_accurate("bf16", got[0] * (1 + 2.0 ** -7), got[1], ref[0], ref[1], rows, keys)


@pytest.mark.parametrize("D", DIMS)
def test_the_check_of_weights_tells_fp32_from_bf16(D):
    Q, K, _, _, _ = inputs(D)
    L, scale = LENS[0], 1 / np.sqrt(D)
    rows = A.score_rms(Q[:1], K[:1], None, [L])

    def added(t, q, k):
        s = np.stack([(k[0, h // (H // G), :L].astype(t) @ q[0, h].T.astype(t)) * t(scale)
                      for h in range(H)])
        return np.exp(s - t(np.log(L))).sum((0, 2), dtype=t)

    want = added(np.float64, Q, K)
    tol = A.weights_tol(rows, H * T)
    assert A.out_error(added(np.float32, Q, K), want) <= tol
    assert A.out_error(added(np.float64, bf16(Q), bf16(K)), want) > 10 * tol
