"""Strided arrays of the HIP wrapper, without a GPU: memory that only the calls taking strides may
reach.  The HIP runtime is a recorder here, so that a copy that should not happen is seen."""
import numpy as np
import pytest

ADDR = 0x7F0000000000


@pytest.fixture
def hip_rt(monkeypatch):
    import hip_rt
    done = []

    class Recorder:
        def hipMemcpy(self, dst, src, nbytes, kind):
            done.append(("copy", nbytes))
            return 0

        def hipMemset(self, dst, value, nbytes):
            done.append(("set", nbytes))
            return 0

    monkeypatch.setattr(hip_rt, "hip", Recorder)
    hip_rt.done = done
    yield hip_rt
    del hip_rt.done


LAYOUTS = [((2, 3, 4, 3), (60, 20, 5, 1)),     # rows padded from 3 to 5 elements
           ((2, 3, 4, 8), (96, 8, 24, 1)),     # [batch][rows][heads][D]
           ((2, 3, 4, 8), (0, 32, 8, 1))]      # one batch repeated


@pytest.mark.parametrize("shape,strides", LAYOUTS)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "i32"])
def test_strided_arrays_have_no_contiguous_image(hip_rt, shape, strides, dtype):
    a = hip_rt.DeviceArray.wrap(ADDR, shape, dtype, strides)
    for call in (lambda: a.upload(np.zeros(shape, np.float32)), a.fill_nan, a.bits, a.numpy,
                 lambda: hip_rt.DeviceArray.view(a, 1, (2, 3))):
        with pytest.raises(ValueError):
            call()
    assert not hip_rt.done


def test_contiguous_wraps_are_whole(hip_rt):
    a = hip_rt.DeviceArray.wrap(ADDR, (2, 3), "f32", (3, 1))
    a.upload(np.zeros((2, 3), np.float32))
    a.fill_nan()
    a.bits()
    b = hip_rt.DeviceArray.view(a, 2, (4,))
    assert (b.ptr, b.nbytes) == (ADDR + 8, 16)
    assert hip_rt.done == [("copy", 24), ("set", 24), ("copy", 24)]


def test_calls_without_strides_refuse_strided_tables_and_workspaces(am, monkeypatch):
    """Encoding tables and workspaces reach the library by address alone: ValueError before any
    call of it, as for Q, K, V and the output."""
    import hip_rt

    class Library:
        def __getattr__(self, name):
            return lambda *args: pytest.fail(f"{name} was called")

    monkeypatch.setattr(am, "lib", Library)

    def arr(shape, strides=None):
        return hip_rt.DeviceArray.wrap(ADDR, shape, "f32", strides)

    x, ws = arr((1, 2, 4, 8)), arr((1 << 16,), (2,))
    whole, table = arr((4, 8)), arr((4, 8), (16, 1))
    for call in (lambda: am.attention_ex(x, x, x, x, workspace=ws), lambda: am.sync_status(ws),
                 lambda: am.make_pe("rope", table_a=table), lambda: am.pe_apply_ex(table, x, 4, None),
                 lambda: am.attention_forward_rope_fused(x, x, x, x, whole, table),
                 lambda: am.attention_forward_rope_fused(x, x, x, x, table, whole),
                 lambda: am.attention_forward_separate_rope(x, x, x, x, x, x, whole, table, 8),
                 lambda: am.attention_forward_separate_rope(x, x, x, x, x, x, table, whole, 8),
                 lambda: am.rope_forward(x, x, table, whole, 8, 4),
                 lambda: am.apply_sinusoidal_embeddings(x, whole, table, x, 4),
                 lambda: am.attention_forward_sinusoidal_hybrid(x, x, x, whole, table, x, x),
                 lambda: am.attention_forward_sinusoidal_hybrid(x, x, x, table, whole, x, x),
                 lambda: am.attention_forward_sinusoidal_separate(x, x, x, whole, table, x, x, x),
                 lambda: am.attention_forward_sinusoidal_separate(x, x, x, table, whole, x, x, x)):
        with pytest.raises(ValueError):
            call()


def test_single_elements_take_no_step(am):
    """A column of a table of lengths of one sequence, one sequence's weights, a single cached row:
    contiguous, whatever the stride of their dimensions of one element."""
    import hip_rt

    def arr(shape, dtype, strides):
        return hip_rt.DeviceArray.wrap(ADDR, shape, dtype, strides)

    lens = arr((1,), "i32", (12,))
    weight = arr((1, 2, 4), "f32", (999, 4, 1))
    assert lens.strides is None and weight.strides is None
    kv = arr((1, 2, 4, 8), "bf16", (0, 32, 8, 1))
    assert kv.strides is None
    am.KvCache(kv, kv, lens, seen=lens, weight=weight)
    assert arr((1, 2, 4, 8), "bf16", (0, 64, 8, 1)).strides == (0, 64, 8, 1)
    assert arr((2,), "i32", (12,)).strides == (12,)
