"""Attention over the paged int8 cache where the tokens that have a row's weight have no value: the row is right in terms of itself."""
import numpy as np
import pytest

from test_gpu_kv import Setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,lengths,group", [(128, [(4000, 1)], 2), (64, [(4000, 1), (700, 1)], 2), (192, [(3000, 1)], 2), (256, [(2500, 1)], 2),
                                               (128, [(900, 70)], 1), (64, [(300, 40), (0, 500)], 2), (80, [(1000, 3)], 3)])
@pytest.mark.parametrize("kw", [dict(), dict(cap=40.0), dict(slopes=True)])
@pytest.mark.parametrize("ahead", [5.0, 9.0, 13.0, 18.0, 25.0])
def test_rows_whose_weight_is_on_tokens_of_no_value(hip, dim, lengths, group, kw, ahead):
    """A first token that takes most of every row's weight and whose value is 0, and another such token further on: the result is what the
    others, of little weight, make of theirs. It has to be right in terms of itself. Off: the weights' rounding by 293 of its units (0.29 for
    each of 64 tokens with codes of 127) for a row whose largest element is below 2^25 of them else: 2^-16.8 of that element, for normal values
    with codes of 32 at 2.5 times that of the others 2^-16.8 * 2.5 / 4; the weight of the first token, and with it that of all others, by five roundings
    of a score of 25 and less: 5 * 25 * 1.44 * 2^-24 = 2^-16.5 at the most, as in any sum of floats."""
    rng = np.random.default_rng(int(ahead) * 1000 + dim)
    s = Setup(hip, rng, 1, dim, [(0, o + n) for o, n in lengths])
    k, v = s.normal(s.now, 2)
    k *= np.float32(0.3)
    direction = np.zeros(dim, np.float32)
    direction[::3] = 1
    direction /= np.sqrt((direction ** 2).sum())
    for at, end in zip(s.now[0], s.now[0][1:]):
        for sink, more in ((at, 1.0), (at + (end - at) // 2, 0.9)):
            k[sink], v[sink] = direction * 4, 0
            k[sink] *= np.float32(more)
    s.append(s.now, k, v)
    b = s.batch([n for _, n in lengths], [o + n for o, n in lengths])
    if kw.get("slopes"):
        kw = dict(slopes=np.linspace(0, 0.002, group).astype(np.float32))
    q = (rng.normal(0, 0.3, (b[2], group, dim)) + direction * ahead * dim ** 0.5 / 4).astype(np.float32)
    dkw = dict(kw, slopes=None if kw.get("slopes") is None else hip.to_device(kw["slopes"]))
    got = s.cache.attend(b[3], hip.to_device(q), **dkw).cpu().numpy()
    want, _ = s.model.attend(b[0], b[1], s.table, q, np.zeros(q.shape, np.float32), **kw)
    size = np.sqrt(np.square(want).sum(-1))
    off = np.sqrt(np.square(got - want).sum(-1))
    assert (size > 0).any() and (off <= 2.0 ** -15 * size).all(), (off / np.maximum(size, 1e-30)).max()


@pytest.mark.parametrize("dim,lengths,sinks", [(128, [(0, 1000)] * 4, (0, 640)), (128, [(0, 900), (300, 700), (0, 1200), (64, 1100)], (0, 65)),
                                               (64, [(5000, 1100)], (0, 4500)), (64, [(0, 600), (700, 500)], (3,)), (200, [(1000, 1100)], (0, 1500))])
@pytest.mark.parametrize("kw", [dict(), dict(window=300), dict(slopes=True), dict(cap=40.0)])
def test_rows_whose_weight_is_on_tokens_of_no_value_among_many(hip, dim, lengths, sinks, kw):
    """The same in batches that fill the GPU, two pages at a time or by each wave for itself, up to 95 pages a wave: a sample of the rows."""
    rng = np.random.default_rng(5)
    heads, ahead = 16, 13.0
    s = Setup(hip, rng, heads, dim, [(0, o + n) for o, n in lengths])
    k, v = s.normal(s.now, 2)
    k *= np.float32(0.3)
    direction = np.ones(dim, np.float32) / np.float32(dim ** 0.5)
    for at in s.now[0][:-1]:
        for sink in sinks:
            k[at + sink], v[at + sink] = direction * 4, 0
    s.append(s.now, k, v)
    b = s.batch([n for _, n in lengths], [o + n for o, n in lengths])
    if kw.get("slopes"):
        kw = dict(slopes=np.linspace(0, 0.001, heads).astype(np.float32))
    q = (rng.normal(0, 0.3, (b[2], heads, dim)) + direction * ahead * dim ** 0.5 / 4).astype(np.float32)
    only = {(int(r), int(h)) for r, h in zip(rng.integers(0, b[2], 60), rng.integers(0, heads, 60))}
    dkw = dict(kw, slopes=None if kw.get("slopes") is None else hip.to_device(kw["slopes"]))
    got = s.cache.attend(b[3], hip.to_device(q), **dkw).cpu().numpy()
    want, _ = s.model.attend(b[0], b[1], s.table, q, np.zeros(q.shape, np.float32), only=only, **kw)
    for r, h in only:
        if np.abs(want[r, h]).max() > 0:
            off = np.sqrt(np.square(got[r, h] - want[r, h]).sum() / np.square(want[r, h]).sum())
            assert off <= 2.0 ** -15, (r, h, off)
