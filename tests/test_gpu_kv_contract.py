"""What the contract of the attention over the paged int8 cache says beside its formula: what a row's bits may depend on, and how precise
ordinary rows are."""
import numpy as np
import pytest

from test_gpu_kv import Setup, dev

pytestmark = pytest.mark.gpu


class Sequences:
    """Sequences that are appended to a cache whose memory holds something else before: pages as `order` deals them, codes and scales of
    earlier owners from `garbage`. Their tokens are drawn from their own seeds, so that one is the same in any company."""

    def __init__(self, hip, heads, dim, lengths, seeds, order, garbage, pages=120, width=16):
        torch = hip.torch
        self.hip, self.lengths = hip, lengths
        free = np.random.default_rng(order).permutation(pages)
        table = np.full((len(lengths), width), -1, np.int32)
        at = 0
        for i, (o, n) in enumerate(lengths):
            need = -(-(o + n) // 64)
            table[i, :need] = free[at:at + need]
            at += need
        self.cache = hip.kv_cache(pages, heads, dim)
        gen = torch.Generator(device=hip.device).manual_seed(garbage)
        for t in (self.cache.keys, self.cache.values):
            t.copy_(torch.randint(-128, 128, t.shape, generator=gen, device=hip.device).to(t.dtype))
        for t in (self.cache.key_scales, self.cache.value_scales):
            t.uniform_(0, 1000, generator=gen)
        old, now = ([l[i] for l in lengths] for i in (0, 1))
        rows = [np.random.default_rng(s).normal(0, 1, (2, o + n, heads, dim)).astype(np.float32) for s, (o, n) in zip(seeds, lengths)]
        for counts, upto, cut in ((old, old, lambda r, o, n: r[:, :o]), (now, [o + n for o, n in lengths], lambda r, o, n: r[:, o:])):
            starts = np.concatenate([[0], np.cumsum(counts)])
            self.batch = hip.kv_batch(dev(hip, starts), dev(hip, upto), dev(hip, table), int(starts[-1]))
            k, v = np.concatenate([cut(r, o, n) for r, (o, n) in zip(rows, lengths)], 1)
            if starts[-1]:
                self.cache.append(self.batch, hip.to_device(k), hip.to_device(v))
        self.starts = starts
        self.seeds = seeds

    def attend(self, q_heads, dim, size, **kw):
        q = np.concatenate([np.random.default_rng(100 + s).normal(0, size, (n, q_heads, dim)) for s, (_, n) in zip(self.seeds, self.lengths)])
        return self.cache.attend(self.batch, self.hip.to_device(q.astype(np.float32)), **kw)

    def rows(self, out, i):
        return out[self.starts[i]:self.starts[i + 1]]


SLOPES = np.array([0.0, 0.02, 0.3, -0.01], np.float32)


@pytest.mark.parametrize("dim", [64, 128, 200])
@pytest.mark.parametrize("kw", [dict(), dict(cap=8.0), dict(cap=30.0), dict(window=90), dict(cap=8.0, window=90), dict(slopes=SLOPES),
                                dict(slopes=SLOPES, cap=8.0), dict(cap=8.0, causal=False), dict(slopes=SLOPES, cap=8.0, window=30)])
@pytest.mark.parametrize("lengths", [[(300, 1), (40, 3), (500, 17), (0, 5)], [(700, 1), (63, 1), (130, 1), (5, 1)], [(0, 130), (70, 60), (200, 33), (100, 9)]])
def test_a_row_is_the_same_in_any_company(hip, lengths, kw, dim):
    """The same sequence among other sequences, on other pages of a memory that holds other things: the same bits. (Sizes as many and as
    large, so that a row's tokens are dealt to as many workgroups.)"""
    if kw.get("slopes") is not None:
        kw = dict(kw, slopes=hip.to_device(kw["slopes"]))
    for size in (0.5, 2.0):
        one = Sequences(hip, 2, dim, lengths, [1, 2, 3, 4], 5, 6)
        want = one.attend(4, dim, size, **kw)
        for place in range(2):
            # the first (or the last but one) stays, the others change places, tokens and pages
            stays = (0, 2)[place]
            rest = [i for i in range(4) if i != stays][::-1]
            order = rest[:stays] + [stays] + rest[stays:]
            seeds = [one.seeds[i] if i == stays else 50 + i for i in order]
            for case in range(2):
                other = Sequences(hip, 2, dim, [lengths[i] for i in order], seeds, 20 + case, 30 + case)
                got = other.attend(4, dim, size, **kw)
                assert hip.torch.equal(other.rows(got, stays), one.rows(want, stays)), (size, stays, case)


@pytest.mark.parametrize("dim", [64, 128])
def test_a_row_is_the_same_in_any_company_of_many(hip, dim):
    """In the launch for many rows."""
    lengths = [(0, 900), (64, 700), (100, 800), (0, 650)]
    one = Sequences(hip, 16, dim, lengths, [1, 2, 3, 4], 5, 6)
    want = one.attend(32, dim, 1.5)
    other = Sequences(hip, 16, dim, [lengths[i] for i in (3, 1, 0, 2)], [9, 2, 8, 7], 11, 12)
    assert hip.torch.equal(other.rows(other.attend(32, dim, 1.5), 1), one.rows(want, 1))


def relative(got, want):
    """The error of all rows together in terms of the result."""
    return np.sqrt(np.square(got - want).sum() / np.square(want).sum())


@pytest.mark.parametrize("dim,heads,lengths", [(64, 2, [(0, 200), (100, 60)]), (128, 2, [(0, 200), (100, 60)]), (192, 1, [(0, 200)]), (256, 1, [(0, 200)]),
                                               (40, 1, [(0, 300)]), (128, 2, [(1500, 1), (900, 1)]), (64, 1, [(1500, 1), (900, 2)]), (256, 1, [(1900, 1)])])
@pytest.mark.parametrize("kw", [dict(), dict(cap=15.0), dict(slopes=True), dict(slopes=True, cap=15.0, window=100), dict(causal=False)])
def test_ordinary_rows_are_as_precise_as_sums_of_floats(hip, dim, heads, lengths, kw):
    """All rows of a call together, in terms of the result. Where scores are off independently of each other by d, rows of independent values
    are off by d of themselves. A score t is off by five roundings of 2^-24 |t|, with the root of their number that is 2^-22.8 |t|, its
    weight by 2^-23 more, and by what the rounding of q to units of 2^-22 of its largest element's binade makes of it: 0.29 units times
    scale |k|, for rows whose largest element is in [2, 8] at most 0.29 * 2^-20 * 1.1. |t| is 4 + 6 at most where the weights are
    (normal scores of standard deviation 2, weighted by their exponentials, are around 4). A cap of 15 adds 2 * 15 roundings. Rounding the
    weights to 2^-23 of the page's largest adds 2^-23, 32-bit sums over up to 31 pages 2^-22. Together below 2^-18; a digit of eight bits
    less of q or the weights would make 2^-15 at the least."""
    rng = np.random.default_rng(dim)
    s = Setup(hip, rng, heads, dim, lengths)
    s.append(s.now, *s.normal(s.now, 2))
    q_heads = 2 * heads
    kw = dict(kw)
    if kw.get("slopes"):
        kw["slopes"] = rng.uniform(0.001, 0.05, q_heads).astype(np.float32)
    q = (s.normal(s.now, 1, q_heads)[0] * 2).clip(-7.9, 7.9)
    dkw = dict(kw, slopes=None if kw.get("slopes") is None else hip.to_device(kw["slopes"]))
    got = s.cache.attend(s.now[3], hip.to_device(q), **dkw).cpu().numpy()
    want, _ = s.model.attend(s.now[0], s.now[1], s.table, q, np.zeros(q.shape, np.float32), **kw)
    assert relative(got, want) < 2.0 ** -18
