"""Sampling on the GPU against the definition in 64 bits."""
import numpy as np
import pytest

import tilers_hip as th
from tests import paged as pg

pytestmark = pytest.mark.gpu
D = th.TileDtype


def kept(x, temp, k, p, min_p):
    """Order, weights in that order and which are kept: x in f64, largest first."""
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.lexsort((np.arange(x.size), -x))
    order = order[x[order] > -np.inf]
    if order.size == 0:
        return order, np.zeros(0), np.zeros(0, bool)
    s = x[order]
    w = np.where(s == s[0], 1.0, np.exp(np.minimum((s - s[0]) / max(temp, 1e-300), 0)))
    keep = np.ones(w.size, bool)
    if 0 < k:
        keep &= np.arange(w.size) < k
    if p < 1:
        part = w * keep
        keep &= np.cumsum(part) - part < p * part.sum()
    keep &= w >= min_p
    if not temp > 0:
        keep[:] = False
    keep[0] = True
    return order, w, keep


def plain(x, u, temp=1.0, k=0, p=1.0, min_p=0.0):
    """The token from 64 bits, and every token that 32-bit weights may give.  A weight is a power to
    base 2 of a product in f32 with its rounding put back, so good to 2^-21, and a mass to as much
    of itself; the whole numbers of 2^-40 add half a step for each token: together `eps` of the
    kept mass.  Tokens that a cut by mass or weight leaves out or keeps by less than that may be on
    its other side, which moves the masses by theirs."""
    order, w, keep = kept(x, temp, k, p, min_p)
    if order.size == 0:
        return -1, {-1}
    eps = 2.0 ** -20 + w.size * 2.0 ** -41
    edge = np.zeros(w.size, bool)
    if min_p > 0:
        edge |= np.abs(w - min_p) < eps * min_p
    if p < 1:
        part = w * (np.arange(w.size) < k if k > 0 else 1)
        before = np.cumsum(part) - part
        edge |= (np.abs(before - p * part.sum()) < 2 * eps * part.sum()) & (part > 0)
    edge[0] = False
    by_index = np.argsort(order)
    mass = np.cumsum((w * keep)[by_index])
    target = min(max(u, 0.0), 1.0) * mass[-1]
    at = min(int(np.searchsorted(mass, target, side="right")), mass.size - 1)
    off = 2 * eps * mass[-1] + w[edge].sum()
    low = mass - (w * keep)[by_index]
    may = (low <= target + off) & (mass >= target - off) & (keep | edge)[by_index]
    return int(order[by_index][at]), set(order[by_index][may].tolist())


def run(dev, stream, x, dtype, u, stride=0, **limits):
    rows, vocab = x.shape
    wide = x
    if stride:
        wide = np.full((rows, stride), 1000 if dtype == D.F32 else 0x7000, x.dtype)
        wide[:, :vocab] = x
    out = pg.put(dev, stream, np.full(rows + 4, -77, np.int32))
    dev_limits = {n: pg.put(dev, stream, np.asarray(v, np.int32 if n == "top_k" else np.float32))
                  for n, v in limits.items()}
    th.sample(pg.put(dev, stream, wide), out, rows, vocab, dtype,
              pg.put(dev, stream, np.asarray(u, np.float32)), stride=stride, stream=stream,
              **dev_limits)
    got = out.copy_to_host(stream).view(np.int32)
    assert (got[rows:] == -77).all()
    return got[:rows]


def check(dev, stream, x, dtype, u, stride=0, **limits):
    got = run(dev, stream, x, dtype, u, stride, **limits)
    wide = pg.widen(x, dtype).astype(np.float64)
    names = dict(temperature="temp", top_k="k", top_p="p", min_p="min_p")
    sure = 0
    for r in range(x.shape[0]):
        want, may = plain(wide[r], float(np.float32(u[r])), **{
            names[n]: (int(v[r]) if n == "top_k" else float(np.float32(v[r])))
            for n, v in limits.items()})
        assert got[r] in may, (r, got[r], want, {n: v[r] for n, v in limits.items()})
        sure += got[r] == want
    return got, sure


@pytest.mark.parametrize("dtype", [D.F32, D.BF16, D.F16])
@pytest.mark.parametrize("rows,vocab,stride", [(3, 1, 0), (5, 2, 3), (4, 63, 0), (7, 1000, 1001),
                                               (3, 4097, 0), (6, 50257, 0), (2, 152064, 152065)])
def test_without_limits(dev, stream, dtype, rows, vocab, stride):
    rng = np.random.default_rng(vocab)
    x = pg.narrow(rng.standard_normal((rows, vocab)) * 2.5, dtype)
    u = rng.random(rows)
    _, sure = check(dev, stream, x, dtype, u, stride)
    _, more = check(dev, stream, x, dtype, u, stride, temperature=rng.uniform(0.3, 2.0, rows))
    assert sure + more >= 2 * rows - 1   # (a border is a matter of 2^-20)


@pytest.mark.parametrize("dtype", [D.F32, D.BF16, D.F16])
@pytest.mark.parametrize("rows,vocab", [(24, 50), (40, 3001), (24, 50257), (8, 128256)])
def test_limits(dev, stream, dtype, rows, vocab):
    rng = np.random.default_rng(vocab + 1)
    x = pg.narrow(rng.standard_normal((rows, vocab)) * 2.5, dtype)
    for limits in (["top_k"], ["top_p"], ["min_p"], ["top_k", "top_p"],
                   ["top_k", "top_p", "min_p"]):
        make = dict(top_k=rng.integers(-1, min(vocab + 5, 3000), rows),
                    top_p=rng.uniform(0.0, 1.1, rows), min_p=rng.uniform(0, 0.2, rows))
        _, sure = check(dev, stream, x, dtype, rng.random(rows),
                        temperature=rng.uniform(0.4, 1.5, rows), **{n: make[n] for n in limits})
        assert sure >= rows - 1


@pytest.mark.parametrize("dtype", [D.F32, D.BF16, D.F16])
@pytest.mark.parametrize("rows", [1, 2, 130])
def test_long_rows(dev, stream, dtype, rows):
    """Few long rows without limits are spread over many workgroups, many are not: the same answers
    at parts' borders, with masked parts, infinities, an empty row and any number."""
    rng = np.random.default_rng(rows)
    vocab = 70001
    x = rng.standard_normal((rows, vocab)).astype(np.float32) * 3
    x[0, :50000] = -np.inf if rows != 2 else np.nan
    x[rows - 1, 60000:] = -np.inf
    u = rng.random(rows)
    check(dev, stream, pg.narrow(x, dtype), dtype, u, vocab + 1)
    for end in (0.0, 1.0, 1 - 2.0 ** -24, -2.0, np.nan):
        got = run(dev, stream, pg.narrow(x, dtype), dtype, np.full(rows, end))
        for r in range(rows):
            order, _, _ = kept(pg.widen(pg.narrow(x[r], dtype), dtype).astype(np.float64), 1.0, 0,
                               1.0, 0.0)
            if end == 1.0:
                assert got[r] == order.max()
            elif not end > 0:
                assert got[r] == order.min()
    flat = pg.narrow(np.full((rows, vocab), 3.5), dtype)
    assert (run(dev, stream, flat, dtype, np.ones(rows)) == vocab - 1).all()
    assert (run(dev, stream, flat, dtype, np.zeros(rows)) == 0).all()
    one = np.full((rows, vocab), np.nan if rows == 2 else -np.inf, np.float32)
    y = pg.narrow(one, dtype)
    assert (run(dev, stream, y, dtype, u) == -1).all()
    one[:, 65000] = -np.float32(np.finfo(np.float16).max)
    y = pg.narrow(one, dtype)
    assert (run(dev, stream, y, dtype, u) == 65000).all()
    z = x.copy()
    z[:, [10, 69999]] = np.inf
    got = run(dev, stream, pg.narrow(z, dtype), dtype, np.where(np.arange(rows) % 2, 0.7, 0.3))
    assert np.array_equal(got, np.where(np.arange(rows) % 2, 69999, 10))
    cold = run(dev, stream, pg.narrow(x, dtype), dtype, u, temperature=np.zeros(rows))
    assert np.array_equal(cold, [kept(pg.widen(pg.narrow(r, dtype), dtype).astype(np.float64), 0.0,
                                      0, 1.0, 0.0)[0][0] for r in x])


@pytest.mark.parametrize("vocab", [170001, 300000])
def test_rows_past_the_registers(dev, stream, vocab):
    """Rows that do not stay in registers, with limits and wide ranges of equal logits."""
    rng = np.random.default_rng(vocab)
    x = pg.narrow(rng.standard_normal((6, vocab)) * 2, D.BF16)
    _, sure = check(dev, stream, x, D.BF16, rng.random(6), top_k=np.array([5, 4000, 100000, 0, 1, 50]),
                    top_p=np.array([0.9, 0.5, 0.99, 0.3, 1.0, 0.0]))
    assert sure >= 5
    x = rng.standard_normal((6, vocab)).astype(np.float32)
    _, sure = check(dev, stream, x, D.F32, rng.random(6), vocab + 3,
                    temperature=rng.uniform(0.5, 1.5, 6), min_p=rng.uniform(0, 0.3, 6))
    assert sure >= 5
    x = rng.standard_normal((3, 4 * vocab + 1)).astype(np.float32)   # hundreds of parts
    _, sure = check(dev, stream, x, D.F32, [0.001, 0.4, 0.9995], temperature=[0.5, 1.0, 2.0])
    assert sure == 3


@pytest.mark.parametrize("limits", [{}, dict(top_k=[0] * 3), dict(top_p=[1.0] * 3)])
@pytest.mark.parametrize("vocab", [9000, 40000, 1 << 20, 1 << 23])
def test_masses_past_53_bits(dev, stream, vocab, limits):
    """All alike: sums of that many weights of 1 in steps of 2^-40, to the first, a middle and the
    last token."""
    x = pg.narrow(np.zeros((3, vocab)), D.BF16)
    got = run(dev, stream, x, D.BF16, [0.0, 0.5, 1.0], **limits)
    assert got.tolist() == [0, vocab // 2, vocab - 1]


def test_counts_are_exact(dev, stream):
    """top_k alone has no borders: with a number just below one the token is the kept one of the
    highest index, with zero that of the lowest."""
    rng = np.random.default_rng(5)
    rows, vocab = 64, 20000
    x = pg.narrow(rng.standard_normal((rows, vocab)), D.BF16)   # many equal logits
    k = np.maximum(1, np.exp(rng.uniform(0, np.log(vocab), rows)).astype(int))
    wide = pg.widen(x, D.BF16).astype(np.float64)
    last = run(dev, stream, x, D.BF16, np.full(rows, 1 - 2.0 ** -24), top_k=k)
    first = run(dev, stream, x, D.BF16, np.zeros(rows), top_k=k)
    for r in range(rows):
        order, _, keep = kept(wide[r], 1.0, int(k[r]), 1.0, 0.0)
        # the mass above u = 1 - 2^-24 is that of the last kept tokens: at most the last few
        held = np.sort(order[keep])
        assert first[r] == held[0]
        assert last[r] in held[-max(1, held.size // 1000 + 3):]


@pytest.mark.parametrize("dtype", [D.F32, D.BF16])
@pytest.mark.parametrize("vocab", [5000, 128256])
def test_equal_logits(dev, stream, dtype, vocab):
    """All alike, and two values: cuts go by the index."""
    u = np.array([0.0, 0.25, 0.5, 0.999, 0.3, 0.7])
    x = pg.narrow(np.zeros((6, vocab)), dtype)
    k = np.array([0, vocab // 2, 7, 2500, 1, vocab])
    got = run(dev, stream, x, dtype, u, top_k=k)
    want = [int(a * (b if b > 0 else vocab)) for a, b in zip(np.float32(u).astype(float), k)]
    assert np.abs(got - want).max() <= 1
    got = run(dev, stream, x, dtype, u, top_p=np.full(6, 0.25))
    assert np.abs(got - np.float32(u).astype(float) * vocab * 0.25).max() <= 2
    y = np.zeros((6, vocab), np.float32)
    y[:, 1::2] = -1
    check(dev, stream, pg.narrow(y, dtype), dtype, u, top_k=np.full(6, vocab // 2 + 10))


def test_edges(dev, stream):
    """Temperatures of zero, tiny, infinite and NaN; limits off their ranges; numbers of 1 and NaN;
    masked logits, whole rows of them, infinities and NaN."""
    rng = np.random.default_rng(6)
    low = np.finfo(np.float32).min
    base = rng.standard_normal(300).astype(np.float32)
    base[200] = 9.0

    def one(x, u, **limits):
        return int(run(dev, stream, np.asarray(x, np.float32)[None], D.F32, [u],
                       **{n: [v] for n, v in limits.items()})[0])

    for t in (0.0, -1.0, np.nan, 1e-40, 1e-12):
        assert one(base, 0.7, temperature=t) == 200
    assert one(base, 0.5, temperature=np.inf) == 150            # uniform
    for limits in (dict(top_k=1), dict(top_p=0.0), dict(top_p=-1.0), dict(min_p=1.5),
                   dict(top_p=1e-30)):
        assert one(base, 0.99, **limits) == 200
    free = one(base, 0.37)
    for limits in (dict(top_k=0), dict(top_k=-5), dict(top_k=300), dict(top_k=2**31 - 1),
                   dict(top_p=1.0), dict(top_p=7.0), dict(top_p=np.nan), dict(min_p=-1.0),
                   dict(min_p=np.nan), dict(min_p=0.0)):
        assert one(base, 0.37, **limits) == free
    assert one(base, 1.0) == 299 and one(base, 5.0) == 299
    assert one(base, np.nan) == 0 and one(base, -3.0) == 0
    masked = base.copy()
    masked[:] = -np.inf
    assert one(masked, 0.5) == -1 and one(masked, 0.5, top_k=3, top_p=0.5) == -1
    masked[:] = np.nan
    assert one(masked, 0.5) == -1
    masked[17] = -3.0
    for limits in ({}, dict(top_k=5), dict(top_p=0.3), dict(top_k=2, top_p=0.9, min_p=0.1)):
        assert one(masked, 0.9, **limits) == 17
    lowest = np.full(300, low, np.float32)
    assert one(lowest, 0.5) == 150 and one(lowest, 0.5, top_k=10) == 5
    lowest[33] = 0.0
    assert one(lowest, 0.99) == 33 and one(lowest, 0.99, top_k=10) == 33
    top = base.copy()
    top[[40, 80]] = np.inf
    assert one(top, 0.4) == 40 and one(top, 0.6) == 80 and one(top, 0.6, top_k=1) == 40
    assert one(top, 0.6, top_p=0.4) == 40 and one(top, 0.6, top_k=50, top_p=0.6) == 80
    huge = np.full(300, low, np.float32)
    huge[5] = np.finfo(np.float32).max   # a difference that overflows
    assert one(huge, 0.99, top_k=10, top_p=0.9) == 5
    zeros = np.where(np.arange(300) % 2, 0.0, -0.0)
    assert one(zeros, 0.5) == 150 and one(zeros, 0.0, top_k=2) == 0
    assert one(zeros, 0.9, top_k=2) == 1


def test_number_of_each_row(dev, stream):
    """Every part of [0, 1) reaches its token: a row for each of 64 numbers, eight tokens."""
    x = np.log(np.arange(1, 9) / 36.0).astype(np.float32)
    u = (np.arange(64) + 0.5) / 64
    got = run(dev, stream, np.repeat(x[None], 64, 0), D.F32, u)
    want = np.searchsorted(np.cumsum(np.arange(1, 9)) / 36.0, u, side="right")
    assert np.array_equal(got, want)
