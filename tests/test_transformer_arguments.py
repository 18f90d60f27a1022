"""CPU: arrays that the Python classes of the transformer layers refuse, before the library is called, and those that they take."""
import numpy as np
import pytest

from tensor_amd import capi


class Reached(Exception):
    pass


class NoGpu:
    """A library that says when it is called."""
    device_index = 0

    def __getattr__(self, name):
        raise Reached(name)


def linear(w, s, b=None, **kw):
    return capi.Linear(NoGpu(), weight=w, scale=s, bias=b, **kw)


ONES = np.ones((2, 4, 8), np.int8)


@pytest.mark.parametrize("weight", [ONES * np.int16(200), ONES * np.int64(-129), ONES * np.float32(0.5), ONES * np.float32(np.nan), ONES * np.uint8(128),
                                    np.where(np.arange(64).reshape(2, 4, 8) == 63, 300, 1), ONES * 1e300])
def test_weights_that_are_no_codes(weight):
    with pytest.raises(capi.HipError):
        linear(weight, np.ones((2, 4), np.float32))


@pytest.mark.parametrize("weight", [ONES, ONES * np.int64(-128), ONES * np.float32(127), ONES.tolist(), ONES.astype(bool)])
def test_weights_that_are_codes(weight):
    with pytest.raises(Reached):
        linear(weight, np.ones((2, 4), np.float32))


@pytest.mark.parametrize("shape", [(4, 2), (8,), (2, 4, 1), (2, 2, 2), (1, 8), (2, 3), (4,), ()])
def test_scales_and_biases_of_another_shape(shape):
    with pytest.raises(capi.HipError):
        linear(ONES, np.ones(shape, np.float32))
    with pytest.raises(capi.HipError):
        linear(ONES, np.ones((2, 4), np.float32), np.ones(shape, np.float32))


@pytest.mark.parametrize("shape", [(4,), (1, 4)])
@pytest.mark.parametrize("weight", [ONES[0], ONES[:1]])
def test_one_expert_may_leave_its_axis_out(weight, shape):
    with pytest.raises(Reached):
        linear(weight, np.ones(shape, np.float32), np.ones(shape, np.float32))


def test_batches_of_another_gpu():
    """What a batch points to is memory of its library's GPU."""
    class Gpu:
        class native:
            kv_append = kv_read = kv_attend = lambda *args: "called"

        def __init__(self, device_index):
            self.device_index = device_index

    cache, batch = object.__new__(capi.KvCache), object.__new__(capi.KvBatch)
    cache.L, cache._cp, batch._bp = Gpu(0), 0, 0
    for call in (lambda: cache.append(batch, None, None), lambda: cache.read(batch), lambda: cache.attend(batch, None)):
        batch.L = Gpu(1)
        with pytest.raises(capi.HipError):
            call()
        batch.L = Gpu(0)
        call()


def test_a_layer_is_made_on_its_librarys_gpu():
    """Whatever GPU is the current one."""
    from contextlib import contextmanager
    current = [0]

    class Gpu(NoGpu):
        device_index = 1

        class torch:
            class cuda:
                @staticmethod
                @contextmanager
                def device(index):
                    current.append(index)
                    yield
                    current.pop()

        class lib:
            @staticmethod
            def otter_hip_linear_create(*args):
                made_on.append(current[-1])
                return 0

        def _check(self, rc):
            assert rc == 0

    made_on = []
    capi.Linear(Gpu(), weight=ONES, scale=np.ones((2, 4), np.float32))
    assert made_on == [1] and current == [0]
