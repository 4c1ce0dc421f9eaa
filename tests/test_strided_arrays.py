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
