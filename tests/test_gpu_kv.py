"""The paged int8 cache of keys and values: tokens into it, out of it and attention over it, against numpy in 64 bits. Codes and
scales have to be the same numbers; the bound on attention is worked out beside the model (transformer_model.Cache.attend)."""
import ctypes as C

import numpy as np
import pytest

from tensor_amd import capi
from transformer_model import BLOCK, Cache

pytestmark = pytest.mark.gpu


def dev(hip, a, dtype=np.int32):
    return hip.to_device(np.asarray(a, dtype))


class Setup:
    """A cache on the GPU and its model, with a page table in no order. `lengths`: (tokens before, tokens that come)."""

    def __init__(self, hip, rng, heads, dim, lengths, *, front=0, behind=0, spare=3):
        self.hip, self.rng, self.heads, self.dim = hip, rng, heads, dim
        need = [-(-(o + n) // BLOCK) for o, n in lengths]
        self.pages = sum(need) + spare
        order = rng.permutation(self.pages)
        self.table = np.full((len(lengths), max(need + [1])), -1, np.int32)
        at = 0
        for i, k in enumerate(need):
            self.table[i, :k] = order[at:at + k]
            at += k
        self.model, self.cache = Cache(self.pages, heads, dim), hip.kv_cache(self.pages, heads, dim)
        for t in (self.cache.keys, self.cache.values):  # nothing has to be cleared
            t.copy_(hip.torch.randint(-128, 128, t.shape, device=hip.device).to(t.dtype))
        self.cache.key_scales.fill_(float("nan")), self.cache.value_scales.fill_(float("nan"))
        self.before = self.batch([o for o, _ in lengths], [o for o, _ in lengths])
        self.now = self.batch([n for _, n in lengths], [o + n for o, n in lengths], front, behind)
        self.append(self.before, *self.normal(self.before, 2))

    def batch(self, counts, lengths, front=0, behind=0):
        starts = (front + np.concatenate([[0], np.cumsum(counts)])).astype(np.int32)
        lengths = np.asarray(lengths, np.int32)
        rows = int(starts[-1]) + behind
        b = self.hip.kv_batch(dev(self.hip, starts), dev(self.hip, lengths), dev(self.hip, self.table), rows)
        return starts, lengths, rows, b

    def normal(self, batch, k, heads=None):
        return [self.rng.normal(0, 1 + i, (batch[2], heads or self.heads, self.dim)).astype(np.float32) for i in range(k)]

    def append(self, batch, k, v):
        self.cache.append(batch[3], self.hip.to_device(k), self.hip.to_device(v))
        self.model.append(batch[0], batch[1], self.table, k, v)

    def check_read(self, batch):
        into = self.normal(batch, 2)
        got = [self.hip.to_device(t) for t in into]
        self.cache.read(batch[3], *got)
        for g, w in zip(got, self.model.read(batch[0], batch[1], self.table, into)):
            np.testing.assert_array_equal(g.cpu().numpy(), w)

    def check_attend(self, batch, q, **kw):
        into = self.rng.normal(0, 1, q.shape).astype(np.float32)
        out = self.hip.to_device(into)
        dkw = dict(kw, slopes=None if kw.get("slopes") is None else self.hip.to_device(kw["slopes"]))
        self.cache.attend(batch[3], self.hip.to_device(q), out=out, **dkw)
        want, bound = self.model.attend(batch[0], batch[1], self.table, q, into, **kw)
        check_close(out.cpu().numpy(), want, bound)


def check_close(got, want, bound):
    nan = np.isnan(want)
    np.testing.assert_array_equal(np.isnan(got), nan)
    off = np.where(nan, 0, np.abs(np.where(nan, 0, got) - np.where(nan, 0, want)) - bound)
    assert (off <= 0).all(), "worst %g over its bound at %s" % (off.max(), np.unravel_index(off.argmax(), off.shape))


RAGGED = [(0, 1), (0, 64), (63, 1), (64, 1), (1, 63), (5, 200), (0, 0), (130, 65), (128, 128), (10, 0), (0, 129)]


@pytest.mark.parametrize("heads,dim", [(1, 64), (3, 128), (2, 80), (1, 1), (2, 17), (1, 192), (2, 256), (1, 250)])
def test_append_and_read(hip, heads, dim):
    s = Setup(hip, np.random.default_rng(dim), heads, dim, RAGGED, front=2, behind=3)
    s.append(s.now, *s.normal(s.now, 2))
    s.check_read(s.now)
    s.check_read(s.batch(s.now[1], s.now[1], 1, 1))


def test_append_rounds_older_tokens_anew(hip):
    """Tokens one by one, each larger than the last, then a smaller one: the page's scale grows and does not shrink."""
    rng = np.random.default_rng(0)
    s = Setup(hip, rng, 2, 48, [(0, 0), (61, 0)])
    lengths = np.array([0, 61])
    for step in range(8):
        lengths += 1
        b = s.batch([1, 1], lengths)
        k, v = s.normal(b, 2)
        size = np.float32(1.5 ** step if step < 7 else 0.01)
        s.append(b, k * size, v * size)
        s.check_read(s.batch(lengths, lengths))


@pytest.mark.parametrize("dim", [64, 80])
def test_sequences_cut_and_gone_on_from(hip, dim):
    """Tokens taken back, as a draft that was not accepted: the next ones come where the first of them were."""
    s = Setup(hip, np.random.default_rng(dim), 2, dim, [(100, 60), (64, 70), (3, 9), (0, 130)])
    s.append(s.now, *s.normal(s.now, 2))
    for kept, more in ([70, 64, 3, 129], [5, 1, 2, 1]), ([1, 64, 0, 63], [9, 66, 1, 2]):
        b = s.batch(more, [n + m for n, m in zip(kept, more)])
        s.append(b, *s.normal(b, 2))
        s.check_read(s.batch([n + m for n, m in zip(kept, more)], [n + m for n, m in zip(kept, more)]))
        s.check_attend(b, s.normal(b, 1, 4)[0])


def test_append_of_ties_zeros_and_what_is_not_finite(hip):
    rng = np.random.default_rng(1)
    s = Setup(hip, rng, 2, 64, [(0, 70), (3, 40), (0, 5), (0, 64)])
    k, v = s.normal(s.now, 2)
    k[:64] = rng.integers(-254, 255, (64, 2, 64)).astype(np.float32) / 2  # ties: with 127 in the page its scale is 1
    k[0, :, 0] = 127
    k[64:, 0, 3] = np.inf
    v[:, :, 7] = np.nan
    v[70:75, 1, 9] = -np.inf
    a, b = s.now[0][2], s.now[0][3]
    k[a:b], v[a:b] = 0, np.float32(1e-35)                                # below the least scale
    v[s.now[0][3]:] *= np.float32(2.0 ** 120)
    k[s.now[0][3]:] *= np.float32(2.0 ** -90)
    s.append(s.now, k, v)
    s.check_read(s.now)


def test_rounding_is_that_of_the_exact_quotient(hip):
    """Values at, right below and right above the middle between two codes, for scales of every mantissa."""
    rng = np.random.default_rng(2)
    heads, dim = 16, 256
    s = Setup(hip, rng, heads, dim, [(0, 64)] * 8)
    k, v = s.normal(s.now, 2)
    for x in (k, v):
        for i in range(8):
            for h in range(heads):
                page = x[64 * i:64 * i + 64, h]
                most = np.float32(rng.uniform(1, 2) * 2.0 ** rng.integers(-60, 60))
                sc = np.float32(np.float64(most) / 127)
                mid = ((rng.integers(-127, 127, page.shape) + 0.5) * np.float64(sc)).astype(np.float32)
                page[:] = np.nextafter(mid, mid * rng.choice([-1, 1, 2], page.shape).astype(np.float32))
                page[np.abs(page) > most] = 0
                page[0, 0] = most
    s.append(s.now, k, v)
    s.check_read(s.now)


def test_batches_that_say_too_much(hip):
    """More rows than tokens, pages that are none, a table that is too short, sequences without tokens."""
    rng = np.random.default_rng(3)
    s = Setup(hip, rng, 2, 64, [(0, 100), (0, 200), (0, 70)], front=1, behind=2)
    s.append(s.now, *s.normal(s.now, 2))
    s.table[1, 1], s.table[2, 0] = s.pages, -7
    counts = [100, 200, 70]
    for lengths in ([60, 200, 70], [100, 260, 70], [0, 200, 5], [100, 100000, 70]):
        b = s.batch(counts, lengths, 1, 2)
        s.append(b, *s.normal(b, 2))
        s.check_read(b)
        if max(lengths) < 1000:
            s.check_attend(b, s.normal(b, 1, 4)[0])
            s.check_attend(b, s.normal(b, 1, 4)[0], causal=False, window=50)


@pytest.mark.parametrize("heads,group,dim", [(1, 1, 64), (2, 4, 128), (3, 1, 80), (1, 7, 96), (1, 16, 32), (2, 2, 1), (1, 5, 17), (1, 2, 192),
                                             (2, 3, 256), (1, 33, 64)])
def test_attend(hip, heads, group, dim):
    s = Setup(hip, np.random.default_rng(heads * dim + group), heads, dim, RAGGED, front=3, behind=2)
    s.append(s.now, *s.normal(s.now, 2))
    s.check_attend(s.now, s.normal(s.now, 1, heads * group)[0] * 2)


@pytest.mark.parametrize("kw", [dict(causal=False), dict(window=1), dict(window=70), dict(window=64, causal=False), dict(cap=3.0),
                                dict(cap=50.0, window=100), dict(slopes=True), dict(slopes=True, causal=False), dict(scale=0.7),
                                dict(scale=0.0), dict(scale=-1.0), dict(cap=20.0, slopes=True, window=90)])
@pytest.mark.parametrize("dim", [64, 128])
def test_attend_options(hip, kw, dim):
    rng = np.random.default_rng(7)
    s = Setup(hip, rng, 2, dim, RAGGED)
    s.append(s.now, *s.normal(s.now, 2))
    if kw.get("slopes"):
        kw = dict(kw, slopes=rng.uniform(0.01, 0.5, 6).astype(np.float32))
    s.check_attend(s.now, s.normal(s.now, 1, 6)[0], **kw)


@pytest.mark.parametrize("kw", [dict(), dict(causal=False), dict(cap=4.0), dict(cap=60.0, window=200), dict(cap=8.0, causal=False)])
@pytest.mark.parametrize("dim", [40, 64, 128])
def test_slopes_of_every_kind(hip, dim, kw):
    """None, slight and steep ones, such as grow with the distance, on pages in front of the rows, around them and behind them."""
    rng = np.random.default_rng(dim)
    s = Setup(hip, rng, 2, dim, [(600, 70), (0, 300), (63, 1), (129, 1), (448, 16)])
    s.append(s.now, *s.normal(s.now, 2))
    slopes = np.array([0, 0.001, 0.7, 3.0, -0.02, 0.25], np.float32)
    s.check_attend(s.now, s.normal(s.now, 1, 6)[0], slopes=slopes, **kw)


@pytest.mark.parametrize("dim", [64, 128])
def test_slopes_beyond_all_measure(hip, dim):
    """A row of them is its own value: every other weight is exp of a million and more below 0."""
    s = Setup(hip, np.random.default_rng(3), 1, dim, [(600, 70), (0, 200), (700, 1)])
    k, v = s.normal(s.now, 2)
    s.append(s.now, k, v)
    q = hip.to_device(s.normal(s.now, 1, 4)[0])
    own = s.cache.read(s.now[3])[1].cpu().numpy()
    for cap in (0.0, 5.0):
        got = s.cache.attend(s.now[3], q, cap=cap, slopes=hip.to_device(np.array([1e6, 1e30, 1e37, 2e38], np.float32))).cpu().numpy()
        # the weight is 1 exactly; the codes' products with it are exact, and scaled by 32-bit numbers, four roundings of 2^-24
        np.testing.assert_allclose(got, np.broadcast_to(own, got.shape), rtol=2.0 ** -21, atol=0)


@pytest.mark.parametrize("dim", [64, 128, 192, 200])
@pytest.mark.parametrize("lengths", [[(2000, 1)], [(3999, 1), (10, 1), (0, 0), (1000, 1)], [(1500, 9)], [(0, 700), (1300, 1)], [(9000, 1)],
                                     [(70, 1), (7000, 2), (0, 1)], [(5000, 40)]])
def test_attend_of_long_caches(hip, dim, lengths):
    """Few rows: the pages go to several workgroups and are joined behind them, or to the waves of one."""
    s = Setup(hip, np.random.default_rng(11), 1, dim, lengths, front=1, behind=1)
    s.append(s.now, *s.normal(s.now, 2))
    for kw in (dict(), dict(window=300), dict(cap=10.0)):
        s.check_attend(s.now, s.normal(s.now, 1, 3)[0], **kw)


@pytest.mark.parametrize("dim,kw", [(128, dict()), (80, dict()), (128, dict(window=300)), (100, dict(causal=False)), (128, dict(cap=5.0)),
                                    (128, dict(slopes=True, cap=30.0)), (64, dict()), (64, dict(slopes=True)), (192, dict()), (256, dict(window=500))])
def test_attend_of_many_rows(hip, dim, kw):
    """Batches that fill the GPU several times, ragged, from one row to 1500 a sequence; a sample of rows, the first and the last of each
    sequence and of some tiles among them, against the model."""
    rng = np.random.default_rng(dim)
    heads = 16
    lengths = [(0, 1500), (300, 1333), (100, 1), (0, 17), (70, 1111), (0, 0), (500, 48), (0, 300)]
    s = Setup(hip, rng, heads, dim, lengths, front=1, behind=2)
    s.append(s.now, *s.normal(s.now, 2))
    q = s.normal(s.now, 1, heads)[0]
    if kw.get("slopes"):
        kw = dict(kw, slopes=rng.uniform(0.01, 0.5, heads).astype(np.float32))
    starts = s.now[0]
    rows = {int(r) for a, b in zip(starts, starts[1:]) if b > a for r in (a, b - 1, a + (b - a) // 64 * 64, max(a, b - 17))} | \
        set(map(int, rng.integers(starts[0], starts[-1], 40)))
    rows = [r for r in rows if starts[0] <= r < starts[-1]]
    only = {(r, int(h)) for r in rows for h in rng.integers(0, heads, 2)}
    into = rng.normal(0, 1, q.shape).astype(np.float32)
    dkw = dict(kw, slopes=None if kw.get("slopes") is None else hip.to_device(kw["slopes"]))
    got = s.cache.attend(s.now[3], hip.to_device(q), out=hip.to_device(into), **dkw).cpu().numpy()
    np.testing.assert_array_equal(got[:1], into[:1])
    np.testing.assert_array_equal(got[-2:], into[-2:])
    want, bound = s.model.attend(starts, s.now[1], s.table, q, into, only=only, **kw)
    r, h = (np.array(t) for t in zip(*sorted(only)))
    check_close(got[r, h], want[r, h], bound[r, h])


@pytest.mark.parametrize("seqs", [64, 65, 150, 4500])
def test_many_sequences(hip, seqs):
    """Up to 64 sequences and beyond, several 64-folds of them; some without rows, some without tokens."""
    rng = np.random.default_rng(seqs)
    most = 140 if seqs < 1000 else 2
    lengths = [(int(rng.integers(0, most)), int(rng.integers(0, most) * rng.integers(0, 2))) for _ in range(seqs)]
    s = Setup(hip, rng, 1, 32, lengths, front=1, behind=1)
    s.append(s.now, *s.normal(s.now, 2))
    s.check_read(s.now)
    s.check_attend(s.now, s.normal(s.now, 1, 1)[0])
    if seqs < 1000:
        s.check_attend(s.now, s.normal(s.now, 1, 3)[0], window=40)


@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("lengths", [[(70 * i, 1) for i in range(20)] + [(300, 90)], [(0, 400), (1000, 30)], [(500, 33), (5, 17), (0, 300)]])
def test_attend_of_few_and_many_rows_together(hip, dim, lengths):
    """Sequences of every kind beside each other, in the launch for many rows and in that for few: which one it is follows from the
    average. Two query heads: 16, 32, 48 rows and 64 at a time; pages in odd numbers; a page in the middle that is none."""
    s = Setup(hip, np.random.default_rng(21 + dim), 1, dim, lengths, front=1, behind=2)
    s.append(s.now, *s.normal(s.now, 2))
    for kw in (dict(), dict(window=130), dict(cap=4.0), dict(causal=False), dict(cap=60.0, slopes=np.array([0.05, 0.3], np.float32))):
        s.check_attend(s.now, s.normal(s.now, 1, 2)[0], **kw)
    s.table[-1, 2] = s.pages
    s.check_attend(s.batch([n for _, n in lengths], [o + n for o, n in lengths], 1, 2), s.normal(s.now, 1, 2)[0])


def test_attend_of_scores_beyond_all_measure(hip):
    """Scores up to 2^30, where the largest takes it all, beside others within rounding of nothing."""
    rng = np.random.default_rng(22)
    for size in (2.0 ** 10, 2.0 ** 18, 2.0 ** 22):
        s = Setup(hip, rng, 1, 128, [(0, 300)])
        k, v = s.normal(s.now, 2)
        s.append(s.now, k, v)
        into = np.zeros((300, 1, 128), np.float32)
        q = (k * np.float32(size)).astype(np.float32)
        out = s.cache.attend(s.now[3], hip.to_device(q), scale=1.0).cpu().numpy()
        values = s.model.read(s.now[0], s.now[1], s.table, (k, v))[1]
        # a token's own key is far ahead of every other's: 128 against at most 60 times `size`
        np.testing.assert_allclose(out, values, rtol=2.0 ** -20, atol=2.0 ** -20 * np.abs(values).max())


def test_pages_of_very_different_size(hip):
    """Value scales from 2^-99 to 2^100 beside each other, zeros among them: a page's share is rounded to the largest share of its step,
    not to the largest scale."""
    rng = np.random.default_rng(23)
    n = 64 * 8
    for dim in (64, 128):
        s = Setup(hip, rng, 1, dim, [(0, n)])
        k, v = s.normal(s.now, 2)
        for i, e in enumerate([0, -99, 3, None, -60, 40, 0, 100]):
            v[64 * i:64 * i + 64] *= np.float32(0 if e is None else 2.0 ** e)
        s.append(s.now, k, v)
        # rows up to the fifth page: nothing larger than the third's is in sight, and bounds are in terms of what is
        b = s.batch([300], [300])
        s.check_attend(b, s.normal(b, 1, 2)[0])
        s.check_attend(b, s.normal(b, 1, 2)[0], window=70)
        s.check_attend(s.now, s.normal(s.now, 1, 2)[0])


def test_attend_with_pages_far_from_each_other(hip):
    """One token of a page outweighs thousands of the others, and the largest score comes first, last and in between: the running
    maximum, and the weights of pages that hold little."""
    rng = np.random.default_rng(12)
    for peak in (0, 700, 1999):
        s = Setup(hip, rng, 1, 64, [(0, 2000)])
        k, v = s.normal(s.now, 2)
        k *= np.float32(0.2)
        k[peak] *= 60
        s.append(s.now, k, v)
        b = s.batch([1], [2000])
        q = np.repeat(k[peak][None], 2, 1).reshape(1, 2, 64) * np.float32(0.12)
        s.check_attend(b, q, scale=1.0)
        s.check_attend(b, -q, scale=1.0)


def test_attend_of_queries_of_every_size(hip):
    rng = np.random.default_rng(13)
    s = Setup(hip, rng, 1, 96, [(90, 14)])
    s.append(s.now, *s.normal(s.now, 2))
    q = s.normal(s.now, 1, 2)[0]
    for r, size in enumerate([0, 1e-38, 1e-30, 1e-20, 1e-3, 1, 1e3, 1e20, 1e37]):
        q[r] = q[r] / np.abs(q[r]).max() * np.float32(size)
    q[9, :, 5] = np.inf
    q[10, 0, 95] = np.nan
    q[11, 1, 0] = -np.inf
    q[12, :, 40] = 1e4  # one element far above the others
    for r in (range(4), range(4, 7), range(9, 14)):
        b = s.batch([14], [104])
        one = np.ones_like(q)
        one[list(r)] = q[list(r)]
        s.check_attend(b, one)
    big = np.ones_like(q)
    big[7:9] = q[7:9]
    s.check_attend(s.now, big, scale=1e-37)


@pytest.mark.parametrize("dim", [64, 128, 192, 256])
def test_queries_at_the_end_of_a_binade(hip, dim):
    """The largest fixed-point numbers and sums there are: every element of a row the same, on either side of where the unit changes, and
    every code of the keys 127 or -127; one row, and enough for the launch of many."""
    for lengths in ([(130, 1)], [(0, 40), (70, 9)]):
        s = Setup(hip, np.random.default_rng(dim), 1, dim, lengths)
        k = np.where(np.arange(s.now[2])[:, None, None] % 2, -1, 1) * np.ones((1, 1, dim))
        s.append(s.before, np.sign(s.normal(s.before, 1)[0][:, :, :1]) * np.ones((1, 1, dim), np.float32), s.normal(s.before, 1)[0])
        s.append(s.now, k.astype(np.float32), s.normal(s.now, 1)[0])
        sizes = np.float32([1, 1.9, 1.99182, 1.99183, 1.99184, 1.992, np.nextafter(np.float32(2), np.float32(0)), 2])
        q = np.ones((s.now[2], 16, dim), np.float32) * np.concatenate([sizes, -sizes])[None, :, None]
        s.check_attend(s.now, q, scale=1 / dim)
        s.check_attend(s.now, q, scale=1 / dim, cap=3.0)


def test_strides_between_rows(hip):
    """Keys, values and queries as slices of one projection's result, at offsets that are no multiple of 16 bytes."""
    rng = np.random.default_rng(14)
    for dim, pad in ((64, 0), (64, 3), (30, 1)):
        s = Setup(hip, rng, 2, dim, [(5, 70), (0, 33)])
        rows, width = s.now[2], 8 * dim + pad
        both = hip.to_device(rng.normal(0, 1, (rows, width)).astype(np.float32))
        q = both[:, pad:pad + 4 * dim].unflatten(1, (4, dim))
        k, v = (both[:, pad + o * dim:pad + (o + 2) * dim].unflatten(1, (2, dim)) for o in (4, 6))
        s.cache.append(s.now[3], k, v)
        s.model.append(s.now[0], s.now[1], s.table, k.cpu().numpy(), v.cpu().numpy())
        s.check_read(s.now)
        want, bound = s.model.attend(s.now[0], s.now[1], s.table, q.cpu().numpy(), np.zeros((rows, 4, dim), np.float32))
        check_close(s.cache.attend(s.now[3], q).cpu().numpy(), want, bound)


def test_results_do_not_hang_on_the_rest_of_the_batch(hip):
    """The same bits again, alone or beside others where the workgroups of a row are as many, and with another order of pages."""
    rng = np.random.default_rng(15)
    s = Setup(hip, rng, 2, 128, [(300, 1), (40, 3), (500, 17)])
    s.append(s.now, *s.normal(s.now, 2))
    q = hip.to_device(s.normal(s.now, 1, 8)[0])
    out = s.cache.attend(s.now[3], q)
    for _ in range(3):
        assert hip.torch.equal(out, s.cache.attend(s.now[3], q))


def test_decoding_steps_on_a_stream_and_replayed(hip):
    """append and attend as a decoder calls them, token by token, on a stream of its own; then captured once and replayed with lengths
    and pages that change in place."""
    torch = hip.torch
    rng = np.random.default_rng(16)
    steps, seqs, heads, dim = 70, 3, 2, 64
    s = Setup(hip, rng, heads, dim, [(20, steps), (0, steps), (1000, steps)])
    old = np.array([20, 0, 1000])
    tokens = [[rng.normal(0, 1, (seqs, n, dim)).astype(np.float32) for n in (heads, heads, 2 * heads)] for _ in range(steps)]
    wants = []
    for t in range(steps):
        lengths = old + t + 1
        starts = np.arange(seqs + 1, dtype=np.int32)
        s.model.append(starts, lengths, s.table, tokens[t][0], tokens[t][1])
        wants.append(s.model.attend(starts, lengths, s.table, tokens[t][2], np.zeros((seqs, 2 * heads, dim), np.float32)))
    lengths = dev(hip, old)
    batch = hip.kv_batch(dev(hip, np.arange(seqs + 1)), lengths, dev(hip, s.table), seqs)
    k, v, q = (hip.to_device(t) for t in tokens[0])
    out = torch.empty_like(q)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def step():
        lengths.add_(1)
        s.cache.append(batch, k, v)
        s.cache.attend(batch, q, out=out)

    graph = None
    with torch.cuda.stream(stream):
        for t in range(steps):
            for to, a in zip((k, v, q), tokens[t]):
                to.copy_(torch.from_numpy(a))
            if t < 20:
                step()
            else:
                if graph is None:
                    stream.synchronize()
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph, stream=stream):
                        step()
                graph.replay()
            stream.synchronize()
            check_close(out.cpu().numpy(), *wants[t])
            hip.empty(1 << 16, np.float32).zero_()


def test_recorded(hip):
    """append, read and attend through otter_hip_record_begin / _end, replayed."""
    rng = np.random.default_rng(17)
    s = Setup(hip, rng, 1, 64, [(1500, 2), (10, 70)])
    kn, vn = s.normal(s.now, 2)
    qn = s.normal(s.now, 1, 4)[0]
    s.model.append(s.now[0], s.now[1], s.table, kn, vn)
    k, v, q = (hip.to_device(t) for t in (kn, vn, qn))
    out, ko, vo = (hip.torch.zeros_like(t) for t in (q, k, v))
    work = hip.empty(1 << 22, np.int8)
    stream, rec = C.c_void_p(), C.c_void_p()
    hip.torch.cuda.synchronize()
    L = hip.lib
    hip._check(L.otter_hip_record_begin(C.byref(stream)))
    a, b = C.byref(s.cache.args), C.byref(s.now[3].args)
    d = C.byref(capi.KvAttendDesc(4, 64 ** -0.5, 0.0, 1, 0, None))
    size = C.c_size_t
    hip._check(L.otter_hip_kv_append(a, b, hip.ptr(k), size(64), hip.ptr(v), size(64), stream))
    hip._check(L.otter_hip_kv_read(a, b, hip.ptr(ko), hip.ptr(vo), stream))
    hip._check(L.otter_hip_kv_attend(a, b, d, hip.ptr(q), size(256), hip.ptr(out), hip.ptr(work), size(1 << 22), stream))
    hip._check(L.otter_hip_record_end(stream, C.byref(rec)))
    want, bound = s.model.attend(s.now[0], s.now[1], s.table, qn, np.zeros(qn.shape, np.float32))
    keys, values = s.model.read(s.now[0], s.now[1], s.table, (kn, vn))
    for _ in range(3):
        for t in (out, ko, vo):
            t.zero_()
        hip._check(L.otter_hip_record_launch(rec, hip.stream()))
        hip.torch.cuda.synchronize()
        check_close(out.cpu().numpy(), want, bound)
        np.testing.assert_array_equal(ko.cpu().numpy(), keys)
        np.testing.assert_array_equal(vo.cpu().numpy(), values)
    hip._check(L.otter_hip_record_destroy(rec))


def test_a_cache_over_4_gib(hip):
    """Pages at offsets that pass 32 bits."""
    rng = np.random.default_rng(18)
    heads, dim = 8, 256
    page = heads * 4 * 4096
    pages = (5 << 30) // page
    cache = hip.kv_cache(pages, heads, dim)
    table = np.array([[pages - 1, 2, pages - 2]], np.int32)
    model = Cache(3, heads, dim)
    small = np.array([[0, 1, 2]], np.int32)
    n = 150
    starts, lengths = np.array([0, n], np.int32), np.array([n], np.int32)
    b = hip.kv_batch(dev(hip, starts), dev(hip, lengths), dev(hip, table), n)
    k, v = (rng.normal(0, 1, (n, heads, dim)).astype(np.float32) for _ in range(2))
    cache.append(b, hip.to_device(k), hip.to_device(v))
    model.append(starts, lengths, small, k, v)
    for got, want in zip(cache.read(b), model.read(starts, lengths, small, (k, v))):
        np.testing.assert_array_equal(got.cpu().numpy(), want)
    q = rng.normal(0, 1, (n, heads, dim)).astype(np.float32)
    want, bound = model.attend(starts, lengths, small, q, np.zeros(q.shape, np.float32))
    check_close(cache.attend(b, hip.to_device(q)).cpu().numpy(), want, bound)


def test_refusals_of_the_binding(hip):
    torch = hip.torch
    cache = hip.kv_cache(4, 2, 64)
    i = [dev(hip, [0, 3]), dev(hip, [3]), dev(hip, [[0]])]
    b = hip.kv_batch(*i, 3)
    good = torch.zeros((3, 2, 64), device=hip.device)
    for bad in (good.cpu(), good.double(), good[:2], good[:, :1], good.transpose(0, 1), good.expand(3, 2, 64)[..., ::2], None):
        with pytest.raises(capi.HipError):
            cache.append(b, bad, good)
        with pytest.raises(capi.HipError):
            cache.append(b, good, bad)
    for bad in (good[:2], good.half(), torch.zeros((3, 3, 64), device=hip.device), good[..., :32]):
        with pytest.raises(capi.HipError):
            cache.attend(b, bad)
    with pytest.raises(capi.HipError):
        cache.attend(b, good, slopes=torch.zeros(3, device=hip.device))
    with pytest.raises(capi.HipError):
        cache.attend(b, good, out=good[:2])
    for kw in (dict(cap=-1.0), dict(scale=float("nan")), dict(window=-1), dict(cap=float("inf"))):
        with pytest.raises(capi.HipError):
            cache.attend(b, good, **kw)
    for args in ((i[0].long(), i[1], i[2]), (i[0][:1], i[1], i[2]), (i[0], i[1], i[2][0]), (i[0].cpu(), i[1], i[2])):
        with pytest.raises(capi.HipError):
            hip.kv_batch(*args, 3)
    for args in ((0, 2, 64), (4, 0, 64), (4, 2, 0), (4, 2, 257)):
        with pytest.raises(capi.HipError):
            hip.kv_cache(*args)
    with pytest.raises(capi.HipError):
        hip.kv_batch(*i, -1)


def test_refusals_of_workspaces_and_of_sizes_beyond_32_bits(hip):
    torch = hip.torch
    cache = hip.kv_cache(1024, 1, 64)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=hip.device)
    starts, lengths, pages = i32(0, 1), i32(60000), torch.arange(1024, dtype=torch.int32, device=hip.device)[None]
    batch = hip.kv_batch(starts, lengths, pages, 1)
    q = torch.zeros((1, 1, 64), device=hip.device)
    wide = torch.zeros((1 << 20, 2), device=hip.device)
    for workspace in (torch.zeros(1 << 20), wide[:, 0], torch.zeros(4, device=hip.device)):
        with pytest.raises(capi.HipError):
            cache.attend(batch, q, workspace=workspace)
    layer = hip.linear(weight=np.ones((16, 64), np.int8), scale=np.ones(16, np.float32))
    for workspace in (torch.zeros(1 << 20), wide[:, 0], torch.zeros(4, device=hip.device)):
        with pytest.raises(capi.HipError):
            layer.forward(wide[:4].reshape(-1, 1).expand(8, 64)[:, :64].contiguous(), workspace=workspace)
    layer.close()
    for n in (-1, 2 ** 31, 2 ** 32 + 1):
        with pytest.raises(capi.HipError):
            hip.kv_batch(starts, lengths, pages, n)


def test_nothing_to_do(hip):
    cache = hip.kv_cache(4, 2, 64)
    none = hip.torch.zeros((0, 2, 64), device=hip.device)
    for b in (hip.kv_batch(dev(hip, [0]), dev(hip, []), dev(hip, np.zeros((0, 1))), 0), hip.kv_batch(dev(hip, [0, 0]), dev(hip, [0]), dev(hip, [[0]]), 0)):
        cache.append(b, none, none)
        assert cache.read(b)[0].shape == none.shape and cache.attend(b, none).shape == none.shape
    b = hip.kv_batch(dev(hip, [0]), dev(hip, []), dev(hip, np.zeros((0, 1))), 2)
    out = hip.torch.full((2, 2, 64), 7.0, device=hip.device)
    assert (cache.attend(b, hip.torch.zeros_like(out), out=out) == 7).all()
