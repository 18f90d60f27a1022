"""Attention over the paged int8 cache with caps far above and far below every score."""
import numpy as np
import pytest

from test_gpu_kv import Setup
from test_gpu_kv_contract import relative

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
def test_caps_beyond_all_measure(hip, dim):
    """A cap far above every score is none, one far below them leaves no differences between them."""
    s = Setup(hip, np.random.default_rng(dim), 2, dim, [(100, 30), (0, 70)])
    s.append(s.now, *s.normal(s.now, 2))
    q = s.normal(s.now, 1, 4)[0]
    slopes = np.array([0.0, 0.01, 0.1, 0.5], np.float32)
    for more in (dict(), dict(slopes=slopes)):
        for cap, same in ((1e6, 1e6), (1e12, 1e6), (1e25, 0.0), (1e30, 0.0), (2e38, 0.0), (1e-3, 1e-3), (1e-20, 1e-20), (1e-36, 1e-36)):
            dkw = {} if not more else dict(slopes=hip.to_device(slopes))
            got = s.cache.attend(s.now[3], hip.to_device(q), cap=cap, **dkw).cpu().numpy()
            want, _ = s.model.attend(s.now[0], s.now[1], s.table, q, np.zeros(q.shape, np.float32), cap=same, **more)
            assert relative(got, want) < 2.0 ** -18, cap


def test_queries_too_large_for_a_low_cap(hip):
    """scale / cap times a large row leaves 32 bits: the scores are the cap, or 0 where a key is 0."""
    s = Setup(hip, np.random.default_rng(3), 1, 64, [(0, 70)])
    k, v = s.normal(s.now, 2)
    k[::3] = 0
    k[5::3] *= np.float32(1e4)
    s.append(s.now, k, v)
    q = (s.normal(s.now, 1, 1)[0] * 1e9).astype(np.float32)
    got = s.cache.attend(s.now[3], hip.to_device(q), cap=1e-36).cpu().numpy()
    want, _ = s.model.attend(s.now[0], s.now[1], s.table, q, np.zeros(q.shape, np.float32), cap=1e-36)
    assert relative(got, want) < 2.0 ** -18
