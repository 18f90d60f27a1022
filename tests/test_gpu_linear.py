"""Int8 products grouped by expert against numpy in 64 bits; the bound is worked out beside the model (transformer_model.linear)."""
import ctypes as C

import numpy as np
import pytest

from tensor_amd import capi
from transformer_model import linear
from test_gpu_kv import check_close, dev

pytestmark = pytest.mark.gpu


def weights(rng, experts, n, k, bias=True):
    w = rng.integers(-127, 128, (experts, n, k)).astype(np.int8)
    return w, rng.uniform(0.5, 1.5, (experts, n)).astype(np.float32) / (75 * k ** 0.5), \
        rng.normal(0, 0.3, (experts, n)).astype(np.float32) if bias else None


def route(rng, experts, counts, x_rows, front=0, behind=0):
    starts = (front + np.concatenate([[0], np.cumsum(counts)])).astype(np.int32)
    return starts, rng.integers(0, x_rows, int(starts[-1]) + behind).astype(np.int32)


def check(hip, rng, x, w, s, b, starts=None, index=None, **kw):
    layer = hip.linear(weight=w, scale=s, bias=b, **kw)
    rows = len(x) if index is None else len(index)
    into = rng.normal(0, 1, (rows, layer.out_features)).astype(np.float32)
    out = hip.to_device(into)
    got = layer.forward(hip.to_device(x), None if starts is None else dev(hip, starts), None if index is None else dev(hip, index), out=out)
    assert got is out
    kw.pop("act_p0", None) if not kw.get("act") else None
    check_close(out.cpu().numpy(), *linear(x, w, s, b, into, starts=starts, index=index, **kw))
    layer.close()


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 33, 64, 100, 129, 300])
@pytest.mark.parametrize("k,n", [(64, 16), (256, 128), (1000, 77), (1, 1), (17, 260), (640, 256)])
def test_one_expert(hip, rows, k, n):
    rng = np.random.default_rng(rows * k + n)
    x = (rng.normal(0, 1, (rows, k)) * rng.uniform(0.1, 10, (rows, 1))).astype(np.float32)
    check(hip, rng, x, *weights(rng, 1, n, k, bias=n != 128))


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("counts", [[1, 0, 0, 2], [0, 0, 0, 0], [5, 16, 17, 40], [100, 3, 0, 200], [0, 300, 0, 0], [64, 64, 128, 256]])
@pytest.mark.parametrize("k,n", [(192, 96), (100, 50)])
def test_experts(hip, counts, gated, k, n):
    rng = np.random.default_rng(sum(counts) + k)
    starts, index = route(rng, 4, counts, 23, front=2, behind=3)
    x = rng.normal(0, 1, (23, k)).astype(np.float32)
    check(hip, rng, x, *weights(rng, 4, 2 * n if gated else n, k), starts, index, gated=gated)


def test_many_experts_and_rows_that_are_none(hip):
    rng = np.random.default_rng(4)
    counts = rng.integers(0, 4, 150) * rng.integers(0, 2, 150)
    starts, index = route(rng, 150, counts, 9)
    index[::5] = 9
    index[1::7] = -1
    index[2::11] = 2 ** 31 - 1
    x = rng.normal(0, 1, (9, 130)).astype(np.float32)
    for gated in (False, True):
        check(hip, rng, x, *weights(rng, 150, 34, 130), starts, index, gated=gated)
    starts = np.minimum(starts, 40)  # rows behind the last expert's stay as they were
    check(hip, rng, x, *weights(rng, 150, 34, 130), starts, index)


def test_rows_in_their_order_by_expert(hip):
    rng = np.random.default_rng(5)
    x = rng.normal(0, 1, (200, 96)).astype(np.float32)
    check(hip, rng, x, *weights(rng, 3, 64, 96), np.array([0, 7, 7, 190], np.int32))
    check(hip, rng, x, *weights(rng, 1, 64, 96), np.array([20, 150], np.int32))


@pytest.mark.parametrize("act,p0", [(1, 0), (2, 0.1), (3, 0), (4, 0), (5, 0)])
@pytest.mark.parametrize("rows", [3, 200])
def test_activations(hip, act, p0, rows):
    rng = np.random.default_rng(act)
    x = rng.normal(0, 6, (rows, 128)).astype(np.float32)
    w, s, b = weights(rng, 1, 100, 128)
    check(hip, rng, x, w, s, b, act=act, act_p0=p0)


def test_rows_of_every_size(hip):
    """Zeros, ties, what is not finite, rows below the least scale and huge ones."""
    rng = np.random.default_rng(6)
    x = rng.normal(0, 1, (12, 256)).astype(np.float32)
    x[0] = 0
    x[1] = rng.integers(-254, 255, 256) / 2
    x[1, 0] = 127
    x[2, 5], x[3, 6], x[3, 7] = np.nan, np.inf, -np.inf
    x[4], x[5] = np.nan, np.inf
    x[6] *= np.float32(1e-32)
    x[7] *= np.float32(1e-28)
    x[8] *= np.float32(1e30)
    x[9, 100] = 1e5
    check(hip, rng, x, *weights(rng, 1, 70, 256))


def test_the_largest_sums(hip):
    """All codes and weights 127: sums at the end of 32 bits."""
    k = 131072
    x, w = np.full((3, k), 2.0, np.float32), np.full((1, 18, k), 127, np.int8)
    x[1] = -2
    w[0, 1] = -127
    check(hip, np.random.default_rng(0), x, w, np.full((1, 18), 1e-4, np.float32), None)


@pytest.mark.parametrize("rows,k,n,kind", [(1, 2048, 2048, 4), (2, 4000, 1030, 4), (1, 32768, 50, 4), (1, 65600, 50, 0), (4, 1000, 300, 4),
                                           (5, 1000, 300, 0), (1, 100, 9000, 0), (16, 250, 40, 4)])
def test_rows_quantized_within_the_launch(hip, rows, k, n, kind):
    """One to sixteen rows, up to what a workgroup's memory holds; values that are not finite among them."""
    rng = np.random.default_rng(rows * k)
    w, s, b = weights(rng, 1, n, k)
    layer = hip.linear(weight=w, scale=s, bias=b)
    assert layer.kernel_kind(rows) == kind
    layer.close()
    x = rng.normal(0, 1, (rows, k)).astype(np.float32)
    check(hip, rng, x, w, s, b)
    x[0, ::7], x[-1, 5], x[-1, k - 1] = 0, np.inf, np.nan
    check(hip, rng, x, w, s, b)


def test_strides(hip):
    rng = np.random.default_rng(7)
    wide = hip.to_device(rng.normal(0, 1, (40, 301)).astype(np.float32))
    w, s, b = weights(rng, 1, 48, 200)
    layer = hip.linear(weight=w[0], scale=s, bias=b)
    for x in (wide[:, 3:203], wide[::2, :200], wide[:1, 100:300].expand(5, 200)):
        xn = x.cpu().numpy()
        check_close(layer.forward(x).cpu().numpy(), *linear(xn, w, s, b, np.zeros((len(xn), 48), np.float32)))
    odd = hip.torch.zeros(20 * 48 + 1, device=hip.device)[1:].view(20, 48)  # a result at an address that is no multiple of 16
    layer.forward(wide[:20, :200], out=odd)
    assert hip.torch.equal(odd, layer.forward(wide[:20, :200]))


def test_a_row_is_the_same_whatever_stands_beside_it(hip):
    rng = np.random.default_rng(8)
    w, s, b = weights(rng, 1, 300, 1000)
    layer = hip.linear(weight=w, scale=s, bias=b)
    x = hip.to_device(rng.normal(0, 1, (700, 1000)).astype(np.float32))
    whole = layer.forward(x)
    for a, e in ((0, 1), (5, 21), (100, 160), (3, 300)):
        assert hip.torch.equal(whole[a:e], layer.forward(x[a:e]))


@pytest.mark.parametrize("kind", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("k,n", [(64, 16), (65, 130), (128, 256), (130, 33), (200, 515), (448, 64), (577, 300), (1000, 270)])
def test_every_launch(hip, kind, k, n):
    """Each launch at sizes that the choice would not give it: outputs and rows that end inside its tiles, steps of inputs in odd and even
    numbers, experts with none, one and many rows, a gate, every activation."""
    rng = np.random.default_rng(kind + k)
    for counts, gated, act in (([1], False, 0), ([300], False, 1), ([0, 130, 0, 129, 1], False, 0), ([70, 0, 65], True, 0), ([128], False, 2),
                               ([257], False, 3), ([40], False, 4), ([33, 31], False, 5), ([64], True, 0)):
        e = len(counts)
        starts, index = route(rng, e, counts, 50, front=2, behind=1)
        x = rng.normal(0, 1, (50, k)).astype(np.float32)
        w, s, b = weights(rng, e, 2 * n if gated else n, k)
        layer = hip.linear(weight=w, scale=s, bias=b, gated=gated, act=act, act_p0=0.1)
        layer.set_kernel(kind)
        assert layer.kernel_kind(5) == kind
        into = rng.normal(0, 1, (len(index), n)).astype(np.float32)
        out = layer.forward(hip.to_device(x), dev(hip, starts), dev(hip, index), out=hip.to_device(into))
        check_close(out.cpu().numpy(), *linear(x, w, s, b, into, starts=starts, index=index, gated=gated, act=act, act_p0=0.1))
        layer.close()


@pytest.mark.parametrize("experts,k,n,rows,gated", [(1, 1000, 1030, 1500, False), (4, 448, 640, 900, True), (3, 320, 1900, 9001, False),
                                                    (2, 130, 1500, 9000, True), (1, 1090, 4100, 4100, False), (1, 64, 8200, 16000, False)])
def test_launches_give_the_same_bits(hip, experts, k, n, rows, gated):
    """Many rows, among them results that are too many for the caches: every launch as the automatic one, bit for bit."""
    torch = hip.torch
    rng = np.random.default_rng(rows)
    w, s, b = weights(rng, experts, 2 * n if gated else n, k)
    layer = hip.linear(weight=w, scale=s, bias=b, gated=gated)
    assert layer.kernel_kind(rows) in (1, 2, 3)
    cuts = np.sort(rng.integers(0, rows + 1, experts - 1))
    starts = dev(hip, np.concatenate([[3], np.maximum(cuts, 3), [rows]]))
    x = hip.to_device(rng.normal(0, 1, (rows // 2, k)).astype(np.float32))
    index = dev(hip, rng.integers(0, rows // 2, rows))
    want = layer.forward(x, starts, index, out=torch.full((rows, n), 5.0, device=hip.device))
    assert (want[:3] == 5).all() and not (want[3:] == 5).any(1).all()
    for kind in range(5):
        layer.set_kernel(kind)
        assert torch.equal(want, layer.forward(x, starts, index, out=torch.full((rows, n), 5.0, device=hip.device)))
    layer.set_kernel(-1)
    with pytest.raises(capi.HipError):
        layer.set_kernel(5)
    layer.close()


def test_a_transformer_layer_replayed(hip):
    """The operators as a layer uses them -- projection, append, attention, projection, experts with a gate, the product behind it --
    eagerly on a stream of its own, then captured and replayed on new inputs."""
    torch = hip.torch
    rng = np.random.default_rng(9)
    heads, group, dim, width, experts, inner, top = 2, 2, 64, 256, 4, 160, 2
    seqs = [(100, 1), (0, 5), (63, 1), (700, 1)]
    rows = sum(n for _, n in seqs)
    mk = lambda *a: weights(rng, *a)
    qkv, proj, up, down = mk(1, (heads * group + 2 * heads) * dim, width), mk(1, width, heads * group * dim), mk(experts, 2 * inner, width), \
        mk(experts, width, inner)
    layers = [hip.linear(weight=w, scale=s, bias=b, gated=g) for (w, s, b), g in ((qkv, False), (proj, False), (up, True), (down, False))]
    from test_gpu_kv import Setup
    s = Setup(hip, rng, heads, dim, seqs)
    batch = s.now
    starts = np.array([0, 5, 5, 11, 2 * rows], np.int32)
    index = rng.permutation(np.repeat(np.arange(rows), top)).astype(np.int32)
    starts_d, index_d = dev(hip, starts), dev(hip, index)
    x = hip.to_device(np.zeros((rows, width), np.float32))

    def layer():
        a = layers[0].forward(x)
        q = a[:, :heads * group * dim].unflatten(1, (heads * group, dim))
        k, v = (a[:, (heads * group + o * heads) * dim:][:, :heads * dim].unflatten(1, (heads, dim)) for o in (0, 1))
        s.cache.append(batch[3], k, v)
        o = s.cache.attend(batch[3], q)
        p = layers[1].forward(o.flatten(1))
        h = layers[2].forward(p, starts_d, index_d)
        return a, o, p, h, layers[3].forward(h, starts_d)

    def check_layer(xn, got):
        """Each operator against the model on what the one before it gave: a scale of rows that differ in the last bit may round another way."""
        a, o, p, h, y = (t.cpu().numpy() for t in got)
        zero = lambda t: np.zeros(t.shape, np.float32)
        check_close(a, *linear(xn, *qkv, zero(a)))
        q = a[:, :heads * group * dim].reshape(rows, heads * group, dim)
        k, v = (a[:, (heads * group + n * heads) * dim:][:, :heads * dim].reshape(rows, heads, dim) for n in (0, 1))
        s.model.append(batch[0], batch[1], s.table, k, v)
        check_close(o, *s.model.attend(batch[0], batch[1], s.table, q, zero(o)))
        check_close(p, *linear(o.reshape(rows, -1), *proj, zero(p)))
        check_close(h, *linear(p, *up, zero(h), starts=starts, index=index, gated=True))
        check_close(y, *linear(h, *down, zero(y), starts=starts))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        inputs = [rng.normal(0, 1, (rows, width)).astype(np.float32) for _ in range(4)]
        x.copy_(torch.from_numpy(inputs[0]))
        got = layer()
        stream.synchronize()
        check_layer(inputs[0], got)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = layer()
        for xn in inputs[1:]:
            x.copy_(torch.from_numpy(xn))
            graph.replay()
            stream.synchronize()
            check_layer(xn, got)
            hip.empty(1 << 16, np.float32).zero_()


def test_refusals_of_the_binding(hip):
    torch = hip.torch
    rng = np.random.default_rng(10)
    w, s, b = weights(rng, 2, 32, 64)
    layer = hip.linear(weight=w, scale=s, bias=b)
    x, starts = torch.zeros((8, 64), device=hip.device), dev(hip, [0, 4, 8])
    assert layer.forward(x, starts).shape == (8, 32)
    for args in ((x,), (x.cpu(), starts), (x.double(), starts), (x[:, :32], starts), (x.t().contiguous().t(), starts), (x, starts.long()),
                 (x, starts[:2]), (x, starts, starts.float()), (x[:0], starts, dev(hip, [0, 0]))):
        with pytest.raises(capi.HipError):
            layer.forward(*args)
    with pytest.raises(capi.HipError):
        layer.forward(x, starts, out=torch.zeros((7, 32), device=hip.device))
    with pytest.raises(capi.HipError):
        layer.forward(x, starts, workspace=hip.empty(16, np.int8))
    assert layer.forward(x[:0], starts).shape == (0, 32)
    for kw in (dict(weight=w[0, 0], scale=s), dict(weight=w, scale=s[:1]), dict(weight=w, scale=s, bias=b[0]), dict(weight=w[:, :31], scale=s[:, :31], gated=True),
               dict(weight=w, scale=s, act=6), dict(weight=w, scale=s, act=1, gated=True), dict(weight=w[:0], scale=s[:0])):
        with pytest.raises(capi.HipError):
            hip.linear(**kw)
    layer.close()
    with pytest.raises(capi.HipError):
        layer.forward(x, starts)


@pytest.mark.parametrize("experts,counts,k,n,gated", [
    (1, [128 * 32 + 1], 64, 4096, False),           # 33 x 16 workgroups: 16 behind a round
    (1, [128 * 37 + 70], 100, 4000, False),         # 96 behind a round, the last with the end of the rows and of the outputs
    (1, [128 * 38 + 3], 64, 4096, False),           # 112: not cut
    (1, [128 * 127 + 128], 130, 2056, True),        # gated, two rounds and 128 blocks of 17
    (5, [1000, 0, 1300, 1, 1930], 192, 4099, False),  # experts of no whole tiles, an odd number of outputs
    (70, [60] * 70, 64, 2100, False)])              # too many experts for their tiles to be counted
def test_workgroups_behind_the_last_whole_round(hip, experts, counts, k, n, gated):
    """The launch of the largest tiles cuts the few that a round of workgroups leaves: the same results as from small tiles, bit by bit."""
    rng = np.random.default_rng(k + n)
    w, s, b = weights(rng, experts, n, k)
    starts, index = route(rng, experts, counts, 300, front=5, behind=4)
    layer = hip.linear(weight=w, scale=s, bias=b, gated=gated)
    x, st, ix = hip.to_device(rng.normal(0, 1, (300, k)).astype(np.float32)), dev(hip, starts), dev(hip, index)
    results = []
    for kind in (1, 3):
        layer.set_kernel(kind)
        out = hip.torch.full((len(index), layer.out_features), 7.5, device=hip.device)
        layer.forward(x, st, ix, out=out)
        results.append(out)
        whole = hip.torch.full((sum(counts), layer.out_features), 7.5, device=hip.device)
        if experts == 1:  # (without `starts` or an index)
            layer.forward(x[ix[5:5 + sum(counts)].long()], out=whole)
            assert hip.torch.equal(whole, out[5:5 + sum(counts)])
    layer.close()
    assert hip.torch.equal(results[0], results[1])
    assert hip.torch.all(results[1][:5] == 7.5) and hip.torch.all(results[1][-4:] == 7.5)
    few = np.r_[5:20, 5 + sum(counts) - 20:5 + sum(counts)]
    experts_of = np.searchsorted(starts, few, side="right") - 1
    xn, got = x.cpu().numpy(), results[1].cpu().numpy()
    for e in set(experts_of.tolist()):
        rows = few[experts_of == e]
        check_close(got[rows], *linear(xn, w[e:e + 1], s[e:e + 1], b[e:e + 1], got[rows], index=index[rows], gated=gated))
