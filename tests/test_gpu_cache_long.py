"""Heads of more than 2^17 rows: eviction that goes through a head's keys in chunks, weights, and
attention, bf16 and fp32."""
import numpy as np
import pytest

import cache_accuracy as A
import cache_helpers as C
from test_gpu_kv_cache import Cache, check_evict, weigh64
from test_gpu_tree_attention import Problem

pytestmark = pytest.mark.gpu

L = (1 << 17) + 77


@pytest.mark.parametrize("budget,recent,kind", [
    (4096, 512, "random"), (L - 5, 7, "random"), (65536, 0, "equal"), (30000, 29000, "few kinds")])
def test_evict(am, dev, budget, recent, kind):
    print(f"[case] evict {budget} {recent} {kind} of {L} rows", flush=True)
    c = Cache(am, "bf16", 1, 2, L + 3, 8, [L], seen=[L + 3])
    rng = np.random.default_rng(2)
    if kind != "random":
        c.weight = np.zeros_like(c.weight) if kind == "equal" else \
            rng.integers(0, 3, c.weight.shape).astype(np.float32)
        c.d_weight.upload(c.weight)
    check_evict(am, c, budget, recent)


@pytest.mark.parametrize("dtype,D", [("bf16", 64), ("f32", 260)])
def test_weights(am, dev, dtype, D):
    import hip_rt
    print(f"[case] weigh {dtype} {D} over {L} rows", flush=True)
    c = Cache(am, dtype, 1, 1, L + 2, D, [L])
    rng = np.random.default_rng(4)
    q, kd, vd = (C.Tensor(rng.standard_normal((1, h, 2, D)), dtype) for h in (4, 1, 1))
    lse = (rng.standard_normal((1, 4, 2)) + np.log(L)).astype(np.float32)
    d = am.Drafts(q.dev, kd.dev, vd.dev)
    am.cache_commit_ex(c.desc, d)
    am.cache_weigh_ex(c.desc, d, C.floats(lse), weight_in=None)
    hip_rt.synchronize()
    K = c.K.numpy()
    want, err = weigh64(q.host, K, lse, None, [2], [L], 1.0 / np.sqrt(D))
    got = c.d_weight.numpy()
    assert (np.abs(got - want) <= 1.01 * err + 10 * C.U32 * want).all()
    assert A.out_error(got, want) <= A.weights_tol(A.score_rms(q.host, K, None, [L + 2]), 8)


@pytest.mark.parametrize("dtype,T,D", [("bf16", 1, 128), ("bf16", 70, 80), ("f32", 3, 64), ("bf16", 2, 300)])
def test_attention(am, dev, dtype, T, D):
    print(f"[case] attention {dtype} {T} {D} over {L} rows", flush=True)
    p = Problem(am, dtype, 1, 2, 1, T, D, L + 2, [L])
    p.run()
    p.check()
    want, want_lse, info = p.want()
    A.attend_accurate(dtype, p.out.numpy(), p.lse.numpy(), want, want_lse,
                      A.score_rms(p.Q.host, p.K.host, p.Kd.host, [L]), info["keys"].max())
