"""The decoding operators' errors as a whole, on the GPU, against their definitions in 64 bits."""
import numpy as np
import pytest

import cache_accuracy as A
import cache_helpers as C
from test_gpu_kv_cache import Cache, weigh64
from test_gpu_tree_attention import Problem

pytestmark = pytest.mark.gpu


def attend(am, dtype, B, Hq, G, T, D, cap, lens, **kw):
    p = Problem(am, dtype, B, Hq, G, T, D, cap, lens, **kw)
    p.run()
    want, want_lse, info = p.want()
    rows = A.score_rms(p.Q.host, p.K.host, p.Kd.host, lens)
    off = A.attend_accurate(dtype, p.out.numpy(), p.lse.numpy(), want, want_lse, rows,
                            info["keys"].max())
    print(f"[case] {dtype} {(B, Hq, G, T, D)} len={lens}: out {off[0]:.3f}, lse {off[1]:.3f} "
          "tolerances", flush=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 65, 80, 96, 100, 128, 130, 160, 192, 200, 256, 257, 264, 384, 500, 512,
                               1000, 1024, 2048, 4100, 8192])
def test_head_sizes(am, dev, dtype, D):
    attend(am, dtype, 2, 4, 2, 3, D, 90, [77, 33], mask="tree", seed=D)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("Hq,G,T,D,lens", [
    (8, 2, 1, 128, [5000, 1]), (8, 1, 3, 64, [3000, 700]), (4, 1, 40, 128, [2900, 40]),
    (6, 2, 60, 96, [1500, 333]), (4, 2, 20, 200, [1999, 64]), (2, 1, 5, 512, [2500, 100]),
    (4, 1, 9, 1024, [1200, 31]), (2, 2, 2, 4096, [700, 650])])
def test_lengths_and_rows(am, dev, dtype, Hq, G, T, D, lens):
    attend(am, dtype, 2, Hq, G, T, D, max(lens) + 5, lens, mask="chain", seed=3)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("Hq,G,T,D,L", [
    (4, 2, 3, 64, 77), (4, 2, 3, 100, 300), (8, 2, 1, 128, 2000), (4, 2, 5, 256, 333),
    (4, 2, 3, 264, 77), (4, 2, 3, 512, 900), (4, 1, 9, 1024, 77), (4, 2, 3, 4100, 60),
    (2, 1, 3, 8192, 600)])
def test_weights(am, dev, dtype, Hq, G, T, D, L):
    import hip_rt
    c = Cache(am, dtype, 1, G, L + T, D, [L])
    rng = np.random.default_rng(D + L)
    q, kd, vd = (C.Tensor(rng.standard_normal((1, h, T, D)) * 1.5, dtype) for h in (Hq, G, G))
    d = am.Drafts(q.dev, kd.dev, vd.dev)
    lse = (rng.standard_normal((1, Hq, T)) + np.log(L)).astype(np.float32)
    am.cache_commit_ex(c.desc, d)
    am.cache_weigh_ex(c.desc, d, C.floats(lse), weight_in=None)
    hip_rt.synchronize()
    K = c.K.numpy()
    want, _ = weigh64(q.host, K, lse, None, [T], [L], 1.0 / np.sqrt(D))
    off = A.out_error(c.d_weight.numpy(), want) / \
        A.weights_tol(A.score_rms(q.host, K, None, [L + T]), Hq // G * T)
    print(f"[case] weigh {dtype} {(Hq, G, T, D, L)}: {off:.3f} tolerances", flush=True)
    assert off <= 1
