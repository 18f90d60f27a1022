"""The launch of the int8 products that keeps the rows' codes in a workgroup's memory, at the end of that memory: 64 KiB, of which the
launch's own statics take 512 bytes. The launch is named before it is made."""
import numpy as np
import pytest

from test_gpu_kv import check_close, dev
from test_gpu_linear import weights
from transformer_model import linear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,k,force,kind", [(2, 32768, -1, 0), (2, 32640, -1, 0), (2, 32512, -1, 4), (2, 32384, -1, 4), (1, 65536, -1, 0), (1, 65409, -1, 0),
                                               (1, 64896, -1, 4), (16, 4096, 4, 0), (16, 3968, 4, 4), (40, 4096, 4, 0), (40, 3968, 4, 4), (4, 16384, 4, 0)])
@pytest.mark.parametrize("gated", [False, True])
def test_codes_that_fill_a_workgroups_memory(hip, rows, k, force, kind, gated):
    rng = np.random.default_rng(rows + k)
    w, s, b = weights(rng, 1, 40, k)
    layer = hip.linear(weight=w, scale=s, bias=b, gated=gated)
    layer.set_kernel(force)
    assert layer.kernel_kind(rows) == kind
    x = rng.normal(0, 1, (rows, k)).astype(np.float32)
    n = layer.out_features
    got = layer.forward(hip.to_device(x)).cpu().numpy()
    check_close(got, *linear(x, w, s, b, np.zeros((rows, n), np.float32), gated=gated))
    layer.close()


def test_sorted_rows_at_the_same_limit(hip):
    rng = np.random.default_rng(0)
    w, s, b = weights(rng, 3, 24, 4096)
    layer = hip.linear(weight=w, scale=s, bias=b)
    x = rng.normal(0, 1, (16, 4096)).astype(np.float32)
    starts, index = np.array([0, 16, 16, 30], np.int32), rng.integers(0, 16, 30).astype(np.int32)
    want = linear(x, w, s, b, np.zeros((30, 24), np.float32), starts=starts, index=index)
    for force in (4, 0):
        layer.set_kernel(force)
        assert layer.kernel_kind(30) == 0
        check_close(layer.forward(hip.to_device(x), dev(hip, starts), dev(hip, index)).cpu().numpy(), *want)
    layer.close()
