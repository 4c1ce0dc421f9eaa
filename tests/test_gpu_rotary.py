"""Rotation by position on the GPU against the definition in float64: pairings, widths, positions far
into a context, strides and alignments, in place and beside other tensors, and the gradient against
the formula's and against differences."""
import numpy as np
import pytest

import cache_helpers as C
import paged_helpers as P

pytestmark = pytest.mark.gpu


def problem(am, dtype, pairing, rot, D, heads, B, T, far, seed=1, amplitude=1.0, order="heads",
            offset=0, pad=0, base=10000.0):
    rng = np.random.default_rng(seed)
    freq, _ = am.rope_frequencies(rot, base)
    pos = rng.integers(0, far + 1, (B, 1)) + np.arange(T)[None]
    xs = [C.Tensor(rng.standard_normal((B, h, T, D)), dtype, order=order, offset=offset, pad=pad)
          for h in heads]
    r = am.Rotary(C.floats(freq), pairing, rot, amplitude)
    return r, xs, pos.astype(np.int32), freq


def close(dtype, got, x, pos, freq, half, rot, amplitude=1.0, inverse=False):
    want, size = P.turned(x, pos, freq, half, rot, amplitude, inverse)
    tol = P.turned_tol(dtype, want, size, pos, freq, amplitude)
    err = np.abs(got - want)
    assert (err <= tol).all(), (np.nanmax(err / tol), np.argwhere(~(err <= tol))[:4].tolist())
    # dims that nothing turns are copied
    assert np.array_equal(got[..., rot:], x[..., rot:])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pairing", ["interleaved", "half"])
@pytest.mark.parametrize("D,rot", [(128, 128), (128, 64), (64, 16), (80, 40), (2, 2), (33, 32), (6, 4),
                                   (100, 50), (257, 256), (1024, 1024), (8192, 8192), (8190, 30)])
def test_sizes(am, dev, dtype, pairing, D, rot):
    r, xs, pos, freq = problem(am, dtype, pairing, rot, D, (3, 1), 2, 5, 1000, amplitude=1.25)
    outs = [C.Tensor(np.full(x.host.shape, 7.0), dtype) for x in xs]
    am.rotary_ex(r, [(x.dev, o.dev) for x, o in zip(xs, outs)], pos=C.ints(pos))
    for x, o in zip(xs, outs):
        close(dtype, o.numpy(), x.host, pos, freq, pairing == "half", rot, 1.25)
        assert np.array_equal(x.numpy(), x.host)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("order", ["heads", "rows"])
@pytest.mark.parametrize("offset,pad", [(0, 0), (8, 8), (1, 0), (0, 1), (3, 5), (4, 4)])
@pytest.mark.parametrize("in_place", [False, True])
def test_strides(am, dev, dtype, order, offset, pad, in_place):
    r, xs, pos, freq = problem(am, dtype, "half", 32, 48, (5,), 3, 7, 50, order=order, offset=offset,
                               pad=pad)
    x = xs[0]
    out = x if in_place else C.Tensor(np.full(x.host.shape, 7.0), dtype, order="heads", offset=2)
    am.rotary_ex(r, [(x.dev, out.dev)], pos=C.ints(pos))
    close(dtype, out.numpy(), x.host, pos, freq, True, 32)


@pytest.mark.parametrize("B,T,heads", [(1, 1, (1,)), (1, 1, (64, 8)), (1, 1000, (2,)), (300, 1, (3, 1)),
                                       (2, 700, (32, 8)), (1, 4097, (1, 1, 1)), (70, 9, (7,))])
def test_tokens(am, dev, B, T, heads):
    r, xs, pos, freq = problem(am, "bf16", "half", 64, 64, heads, B, T, 300)
    am.rotary_ex(r, [(x.dev, x.dev) for x in xs], pos=C.ints(pos))
    for x in xs:
        close("bf16", x.numpy(), x.host, pos, freq, True, 64)


@pytest.mark.parametrize("far", [1 << 20, 1 << 26, (1 << 31) - 100])
def test_far_positions(am, dev, far):
    r, xs, pos, freq = problem(am, "f32", "interleaved", 64, 64, (2,), 4, 6, far, seed=far % 97)
    pos[3] = far + np.arange(6)
    am.rotary_ex(r, [(xs[0].dev, xs[0].dev)], pos=C.ints(pos))
    close("f32", xs[0].numpy(), xs[0].host, pos, freq, False, 64)


def test_negative_and_no_positions(am, dev):
    r, xs, pos, freq = problem(am, "f32", "half", 64, 64, (2, 2), 2, 9, 10)
    pos = -pos - 1
    am.rotary_ex(r, [(xs[0].dev, xs[0].dev)], pos=C.ints(pos))
    close("f32", xs[0].numpy(), xs[0].host, pos, freq, True, 64)
    am.rotary_ex(r, [(xs[1].dev, xs[1].dev)])
    close("f32", xs[1].numpy(), xs[1].host, np.tile(np.arange(9), (2, 1)), freq, True, 64)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_views_of_one_buffer(am, dev, dtype):
    """Queries and keys as columns of a projection's rows, turned where they are."""
    import hip_rt
    rng = np.random.default_rng(5)
    B, T, H, G, D = 2, 11, 6, 2, 32
    row = (H + 2 * G) * D
    x = C.rounded(rng.standard_normal((B, T, H + 2 * G, D)), dtype)
    base = hip_rt.DeviceArray.from_numpy(x, dtype)

    def view(first, n):
        return hip_rt.DeviceArray.wrap(base.ptr + first * D * base.itemsize, (B, n, T, D), dtype,
                                       strides=(T * row, D, row, 1), keep=base)

    freq, _ = am.rope_frequencies(D)
    pos = rng.integers(0, 99, (B, T)).astype(np.int32)
    q, k = view(0, H), view(H, G)
    am.rotary_ex(am.Rotary(C.floats(freq), "half"), [(q, q), (k, k)], pos=C.ints(pos))
    got = base.numpy()
    close(dtype, got[:, :, :H + G].transpose(0, 2, 1, 3),
          x[:, :, :H + G].transpose(0, 2, 1, 3), pos, freq, True, D)
    assert np.array_equal(got[:, :, H + G:], x[:, :, H + G:])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pairing", ["interleaved", "half"])
@pytest.mark.parametrize("D,rot", [(64, 64), (40, 24), (130, 128)])
def test_gradient_formula(am, dev, dtype, pairing, D, rot):
    r, gs, pos, freq = problem(am, dtype, pairing, rot, D, (3,), 2, 6, 5000, seed=9, amplitude=1.1)
    am.rotary_ex(r, [(gs[0].dev, gs[0].dev)], pos=C.ints(pos), inverse=True)
    close(dtype, gs[0].numpy(), gs[0].host, pos, freq, pairing == "half", rot, 1.1, inverse=True)


@pytest.mark.parametrize("pairing", ["interleaved", "half"])
def test_gradient_by_differences(am, dev, pairing):
    """f = sum w y: the inverse rotation of w is (f(x + e) - f(x - e)) / 2 for every unit e (f is
    linear, so the step may be 1)."""
    D, T = 12, 3
    r, xs, pos, freq = problem(am, "f32", pairing, 8, D, (1,), 1, T, 700, seed=4)
    rng = np.random.default_rng(8)
    w = C.Tensor(rng.standard_normal((1, 1, T, D)), "f32")
    g = C.Tensor(np.zeros((1, 1, T, D)), "f32")
    am.rotary_ex(r, [(w.dev, g.dev)], pos=C.ints(pos), inverse=True)
    # every x +- e as a sequence of its own
    n = T * D
    e = np.eye(n).reshape(n, 1, T, D)
    x = C.Tensor(np.concatenate([xs[0].host + e, xs[0].host - e]), "f32")
    y = C.Tensor(np.zeros(x.host.shape), "f32")
    am.rotary_ex(r, [(x.dev, y.dev)], pos=C.ints(np.tile(pos, (2 * n, 1))))
    f = (y.numpy().astype(np.float64) * w.host).sum((1, 2, 3))
    diff = (f[:n] - f[n:]) / 2
    # each of f's terms is off as the rotation is (10 half steps of a pair's size, and its own
    # rounding), x + e by half a step too (through entries of at most 1, two of them)
    _, size = P.turned(np.abs(x.host), np.tile(pos, (2 * n, 1)), freq, pairing == "half", 8)
    per = (np.abs(w.host) * (11 * P.U * size + 3 * P.U * np.abs(x.host).max())).sum((1, 2, 3))
    tol = (per[:n] + per[n:]) / 2 + 12 * P.U * 2 * np.abs(w.host).max()
    assert (np.abs(diff - g.numpy().ravel()) <= tol).all()


def test_inverse_undoes(am, dev):
    r, xs, pos, freq = problem(am, "f32", "half", 128, 128, (4,), 2, 33, 100000)
    p = C.ints(pos)
    y = C.Tensor(np.zeros(xs[0].host.shape), "f32")
    am.rotary_ex(r, [(xs[0].dev, y.dev)], pos=p)
    am.rotary_ex(r, [(y.dev, y.dev)], pos=p, inverse=True)
    _, size = P.turned(xs[0].host, pos, freq, True, 128)
    # two rotations, the first's error through the second (a pair's two entries)
    assert (np.abs(y.numpy() - xs[0].host) <= 3 * 11 * P.U * size).all()


def test_streams_and_captured(am, dev):
    import hip_rt
    r, xs, pos, freq = problem(am, "bf16", "half", 64, 64, (4, 2), 3, 8, 100)
    p = C.ints(pos)
    outs = [C.Tensor(np.zeros(x.host.shape), "bf16") for x in xs]
    call = am.rotary_call(r, [(x.dev, o.dev) for x, o in zip(xs, outs)], pos=p)
    s = hip_rt.Stream()
    g = hip_rt.Graph(s, lambda: call(s))
    for step in range(3):
        now = pos + 17 * step
        p.upload(now)
        g.launch()
        s.synchronize()
        for x, o in zip(xs, outs):
            close("bf16", o.numpy(), x.host, now, freq, True, 64)
        call()  # eager work between the replays
        hip_rt.synchronize()
    g.destroy()
    s.destroy()


@pytest.mark.parametrize("B,T", [(1, 1), (5, 1), (40, 1), (3, 2)])
@pytest.mark.parametrize("order", ["rows", "heads"])
def test_views_of_one_buffer_a_token_each(am, dev, order, B, T):
    """Queries and keys where a projection (or a buffer of heads) holds them, few tokens."""
    import hip_rt
    rng = np.random.default_rng(6)
    H, G, D = 4, 2, 48
    n = H + 2 * G
    x = C.rounded(rng.standard_normal((B, T, n, D) if order == "rows" else (B, n, T, D)), "bf16")
    lie = (0, 2, 1, 3) if order == "rows" else (0, 1, 2, 3)
    base = hip_rt.DeviceArray.from_numpy(x, "bf16")
    s = (n * T * D, D, n * D, 1) if order == "rows" else (n * T * D, T * D, D, 1)
    q, k = (hip_rt.DeviceArray.wrap(base.ptr + 2 * first * s[1], (B, heads, T, D), "bf16", strides=s,
                                    keep=base) for first, heads in ((0, H), (H, G)))
    freq, _ = am.rope_frequencies(D)
    pos = rng.integers(0, 999, (B, T)).astype(np.int32)
    am.rotary_ex(am.Rotary(C.floats(freq), "half"), [(q, q), (k, k)], pos=C.ints(pos))
    got, x = base.numpy().transpose(lie), x.transpose(lie)
    close("bf16", got[:, :H + G], x[:, :H + G], pos, freq, True, D)
    assert np.array_equal(got[:, H + G:], x[:, H + G:])
