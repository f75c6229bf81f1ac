"""The paged cache on the GPU against the plain forms of tests/paged.py: writes and reads exact,
attention within a bound derived from its roundings."""
import ctypes as C

import numpy as np
import pytest

import tilers_hip as th
from tests import paged as pg

pytestmark = pytest.mark.gpu
D = th.TileDtype


# ---- write ---------------------------------------------------------------------------------

def check_write(dev, stream, pool, table, start, length, total_q, src, dtype, stride,
                falling=False):
    """Write src (f32 [2][total_q][heads][D], of dtype's values); every byte of the pool.  Where
    q_start falls a token may be of two sequences, and is then written for one or none: each byte
    is the old or the new one."""
    rows = np.zeros((2, total_q, stride or pool.heads * pool.head_dim), np.float32)
    rows[:, :, :pool.heads * pool.head_dim] = src.reshape(2, total_q, -1)
    k, v = (pg.put(dev, stream, pg.narrow(x, dtype)) for x in rows)
    d = pg.DevicePool(dev, stream, pool)
    old = [x.copy() for x in pool.data]
    seqs = pg.batch(dev, stream, table, start, length, total_q)
    th.kv_cache_write(d.pages, seqs, k, v, dtype, stride, stream)
    for b, n in enumerate(length):
        first, last = (min(max(x, 0), total_q) for x in (start[b], start[b + 1]))
        for i in range(first, last):
            pos = n - (last - first) + i - first
            if pos < 0 or pos // pool.page >= table.shape[1]:
                continue
            page = table[b, pos // pool.page]
            if 0 <= page < pool.num_pages:
                for kv in range(2):
                    pool.put(kv, page, pos % pool.page, src[kv, i])
    for got, want, was in zip(d.codes(), pool.data, old):
        got, want, was = (x.view(np.uint8) for x in (got, want, was))
        assert ((got == want) | ((got == was) & falling)).all()
    for got, want in zip(d.scales(), pool.scale):
        if want is not None and not falling:
            assert np.array_equal(got, want, equal_nan=True)


@pytest.mark.parametrize("cache", [D.BF16, D.F16, D.E4M3, D.I8])
@pytest.mark.parametrize("dtype", [D.BF16, D.F16, D.F32])
@pytest.mark.parametrize("heads,head_dim,page,stride,gap", [
    (2, 128, 16, 0, 0), (8, 64, 32, 8 * 64 + 256, 0), (3, 80, 16, 0, 48), (1, 16, 64, 0, 0),
    (5, 256, 16, 5 * 256 + 8, 16), (2, 192, 16, 0, 0),
])
def test_write(dev, stream, cache, dtype, heads, head_dim, page, stride, gap):
    rng = np.random.default_rng(heads * head_dim + page)
    pool = pg.Pool(rng, cache, 13, page, heads, head_dim, gap, garbage=0x11)
    # a prompt, a step, an idle sequence, a chunk over a page's border, two of odd lengths
    length = [page + 3, 2 * page, 5, page + 2, 1, page - 1]
    new = [page + 3, 1, 0, 5, 1, 2]
    start = np.concatenate([[0], np.cumsum(new)])
    total_q = int(start[-1]) + 3   # rows behind the last sequence
    table = pg.tables(rng, pool, length)
    src = pg.widen(pg.narrow(rng.standard_normal((2, total_q, heads, head_dim)), dtype), dtype)
    check_write(dev, stream, pool, table, start, length, total_q, src, dtype, stride)


@pytest.mark.parametrize("cache", [D.E4M3, D.I8])
def test_write_odd_values(dev, stream, cache):
    """Zeros, infinities, NaN, tiny and huge rows, ties between codes, the largest value alone."""
    rng = np.random.default_rng(3)
    heads, d = 2, 64
    rows = np.zeros((12, heads, d), np.float32)
    rows[1] = rng.standard_normal((heads, d))
    rows[1, 0, 5], rows[1, 1, 6] = np.inf, np.nan
    rows[2, :, 3] = [-np.inf, np.nan]
    rows[3] = 1e-31                       # below the least scale
    rows[4] = rng.standard_normal((heads, d)) * 1e-38
    rows[5] = rng.standard_normal((heads, d)) * 1e37
    rows[6, :, 0] = 3e38
    rows[7] = np.arange(d) - 31.5         # halves: ties of whole numbers once scaled by 127 / 127
    rows[7, :, 0] = 127
    rows[8] = np.linspace(-448, 448, d)   # scaled by one: every binade of e4m3
    rows[9, :, 0], rows[9, :, 1:] = 448, 2.0 ** -9 * (np.arange(1, d) / 4)   # its subnormals
    rows[10] = -0.0
    rows[11] = 1e-30
    src = np.stack([rows, rows[::-1]])
    pool = pg.Pool(rng, cache, 2, 16, heads, d, garbage=0x22)
    check_write(dev, stream, pool, np.array([[1]], np.int32), [0, 12], [12], 12, src, D.F32, 0)


def test_write_any_contents(dev, stream):
    """Lengths and tables that hold anything: what is in range is written, nothing else."""
    rng = np.random.default_rng(4)
    heads, d, page = 2, 64, 16
    pool = pg.Pool(rng, D.I8, 6, page, heads, d, garbage=0x33)
    table = np.array([[0, -1, 6], [2**31 - 1, 1, -2**31], [2, 3, 4], [5, 5, 5]], np.int32)
    start = [0, 20, 22, 60, 90]
    length = [40, 33, 70, 4]   # past the table, into missing pages, fewer than the new tokens
    src = rng.standard_normal((2, 64, heads, d)).astype(np.float32)
    check_write(dev, stream, pool, table, start, length, 64, src, D.F32, 0)
    # falling and negative starts, negative lengths
    pool = pg.Pool(rng, D.I8, 6, page, heads, d, garbage=0x33)
    check_write(dev, stream, pool, table, [-5, 3, 2, 10, 2**31 - 1], [3, 2, -7, 2**31 - 1], 20,
                src[:, :20], D.F32, 0, falling=True)


def test_write_many_sequences(dev, stream):
    rng = np.random.default_rng(5)
    n, page = 201, 16
    pool = pg.Pool(rng, D.BF16, n + 5, page, 1, 16, garbage=0)
    new = rng.integers(0, 3, n)
    start = np.concatenate([[0], np.cumsum(new)])
    length = [int(x) + int(rng.integers(0, 14)) for x in new]
    total = int(start[-1])
    src = pg.widen(pg.narrow(rng.standard_normal((2, total, 1, 16)), D.BF16), D.BF16)
    check_write(dev, stream, pool, pg.tables(rng, pool, [max(1, x) for x in length]), start, length,
                total, src, D.BF16, 0)


# ---- read ----------------------------------------------------------------------------------

@pytest.mark.parametrize("cache", [D.BF16, D.F16, D.E4M3, D.I8])
@pytest.mark.parametrize("dtype", [D.BF16, D.F16, D.F32])
@pytest.mark.parametrize("heads,head_dim,page,gap,max_seq", [
    (2, 128, 16, 0, 150), (4, 64, 64, 0, 131), (1, 80, 32, 16, 100), (3, 256, 16, 0, 40),
    (2, 16, 256, 0, 300),
])
def test_read(dev, stream, cache, dtype, heads, head_dim, page, gap, max_seq):
    rng = np.random.default_rng(heads + head_dim)
    length = [131, 0, 1, page, 40, 150]   # some past max_seq
    pool = pg.Pool(rng, cache, sum(-(-n // page) for n in length) + 2, page, heads, head_dim, gap)
    table = pg.tables(rng, pool, length)
    for b, n in enumerate(length):
        pool.fill(rng, table[b], n)
    table[4, 0] = -1   # a page that was given back reads as zeros
    d = pg.DevicePool(dev, stream, pool)
    seqs = pg.batch(dev, stream, table, [0] * 7, length, 0)
    shape = (len(length), heads, max_seq, head_dim)
    before = np.full(shape, 9, dtype.host_dtype)
    out = [pg.put(dev, stream, before) for _ in range(2)]
    th.kv_cache_read(d.pages, seqs, out[0], out[1], max_seq, dtype, stream)
    for i in range(2):
        want = before.copy()
        for b, n in enumerate(length):
            n = min(n, max_seq)
            # code * scale is exact in f64 and rounds once to f32, then (16 bits) once more
            want[b, :, :n] = pg.narrow(pool.read(i, table[b], n).astype(np.float32), dtype)
        assert np.array_equal(out[i].copy_to_host(stream).reshape(shape), want)


def test_read_past_the_table(dev, stream):
    rng = np.random.default_rng(8)
    pool = pg.Pool(rng, D.E4M3, 3, 16, 1, 16)
    pool.fill(rng, [1, 2], 32)
    d = pg.DevicePool(dev, stream, pool)
    seqs = pg.batch(dev, stream, [[1, 2], [3, 2**31 - 1]], [0, 0, 0], [2**31 - 1, -4], 0)
    out = [pg.put(dev, stream, np.full((2, 1, 50, 16), 9, np.float32)) for _ in range(2)]
    th.kv_cache_read(d.pages, seqs, out[0], out[1], 50, D.F32, stream)
    got = out[0].copy_to_host(stream).reshape(2, 50, 16)
    assert np.array_equal(got[0, :32], pool.read(0, [1, 2], 32)[0].astype(np.float32))
    assert not got[0, 32:].any() and (got[1] == 9).all()


# ---- attention -----------------------------------------------------------------------------

def bound(o, mean, reach, dtype, head_dim, held, codes):
    """How far O may be from 64 bits.  Half a step of a type is u.  O's own rounding: u |o|.  The
    weights' rounding, to dtype or with codes to f16: up sum p |v| at most in the product with V;
    without codes the sum is of the rounded ones too, so the weighted mean moves by
    |sum p e (v - o)| <= up (sum p |v| + |o|).  A score is a sum of D exact products in f32
    (D 2^-24 sum |q k| at most), scaled twice and subtracted (4 roundings of a value of at most 2
    reach log2 e), then a power to base 2 good to 2^-21: weights are off by e each, which moves
    numerator and denominator by as much.  Sums over the positions: held roundings of 2^-24 at
    most, in parts of 8, so 2^-24 (held / 8 + 64).  f16 weights below 2^-14 are multiples of 2^-24
    and the largest is at least 1 (or 1/2 with codes, whose scales are relative to a power of two
    within a factor of two of the largest; values at most that factor, 2, times the largest), a
    position's error 2^-25 of the largest value."""
    u = pg.HALF[dtype]
    up = pg.HALF[D.F16] if codes else u
    e = (head_dim + 8) * 2.0 ** -23 * reach[..., None] + 2.0 ** -20 + 2.0 ** -24 * (held / 8 + 64)
    tol = (up * (mean + (0 if codes else np.abs(o))) + u * np.abs(o)) * 1.01 + 2 * e * mean + 1e-30
    if dtype == D.F16 or codes:
        tol = tol + held * 2.0 ** -24 * (4 if codes else 1) * max(1.0, float(np.abs(mean).max()))
    if dtype == D.F16:
        tol = tol + 2.0 ** -25
    return tol


def run_attention(dev, stream, pool, table, start, length, q, dtype, group, q_stride=0,
                  workspace=None, seqs=None):
    """O of the device for q [total_q][heads][D] (patterns of dtype), guards behind it."""
    total_q, heads, hd = q.shape
    if q_stride:
        wide = np.zeros((total_q, q_stride), q.dtype)
        wide[:, :heads * hd] = q.reshape(total_q, -1)
    else:
        wide = q
    d = pg.DevicePool(dev, stream, pool)
    seqs = seqs or pg.batch(dev, stream, table, start, length, total_q)
    o = pg.put(dev, stream, np.full(q.size + 64, 9, np.uint16))
    room = th.attention_paged_workspace_size(d.pages, seqs, heads)
    ws = dev.alloc(max(1, room // 4), D.F32) if workspace is None else None
    if ws is not None:   # nothing in it is taken for granted
        ws.copy_from_host(np.full(ws.count, np.nan, np.float32), stream)
    th.attention_paged(pg.put(dev, stream, wide), d.pages, seqs, o, heads, dtype, q_stride,
                       ws, room if ws is not None else 0, stream)
    got = o.copy_to_host(stream)
    assert (got[q.size:] == 9).all()
    return got[:q.size].reshape(q.shape)


def check_attention(dev, stream, pool, table, start, length, q, dtype, group, **kw):
    got = run_attention(dev, stream, pool, table, start, length, q, dtype, group, **kw)
    total_q = q.shape[0]
    seen = np.zeros(total_q, bool)
    worst = 0.0
    for b, n in enumerate(length):
        first, last = (min(max(x, 0), total_q) for x in (start[b], start[b + 1]))
        if last <= first:
            continue
        seen[first:last] = True
        held = max(0, min(n, table.shape[1] * pool.page))
        kv = [pool.read(i, table[b], held) for i in range(2)]
        o, mean, reach = pg.attention(pg.widen(q[first:last], dtype).astype(np.float64), kv,
                                      pool.there(table[b], held), last - first, max(n, 0), group)
        tol = bound(o, mean, reach, dtype, pool.head_dim, held, pool.dtype in pg.MOST)
        err = np.abs(pg.widen(got[first:last], dtype) - o)
        bad = ~(err <= tol)
        assert not bad.any(), (b, np.argwhere(bad)[:4], err[bad][:4], tol[bad][:4], o[bad][:4])
        worst = max(worst, float((err / tol).max()) if err.size else 0.0)
    assert (got[~seen] == 9).all()   # rows of no sequence
    return got


def make(rng, cache, dtype, heads, group, head_dim, page, length, new, gap=0, peak=1.0, q_std=1.0,
         extra=0):
    pool = pg.Pool(rng, cache, sum(-(-max(0, n) // page) for n in length) + 2, page, heads,
                   head_dim, gap)
    table = pg.tables(rng, pool, [max(0, n) for n in length])
    for b, n in enumerate(length):
        pool.fill(rng, table[b], n, peak)
    start = np.concatenate([[0], np.cumsum(new)]).tolist()
    q = pg.narrow(rng.standard_normal((start[-1] + extra, heads * group, head_dim)) * q_std, dtype)
    return pool, table, start, q


TYPES = [(D.BF16, D.BF16), (D.F16, D.F16), (D.BF16, D.E4M3), (D.F16, D.E4M3), (D.BF16, D.I8),
         (D.F16, D.I8)]


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("heads,group,head_dim,page", [
    (2, 4, 128, 16), (1, 1, 64, 32), (2, 8, 64, 16), (1, 7, 128, 64), (3, 1, 80, 16),
    (1, 16, 32, 16), (1, 20, 48, 16), (1, 2, 256, 32), (1, 3, 144, 16), (2, 2, 16, 16),
    (1, 71, 64, 16), (1, 3, 112, 64), (1, 5, 208, 16),
])
def test_steps(dev, stream, dtype, cache, heads, group, head_dim, page):
    """Single tokens: from one position to several hundred, pages that end inside a tile."""
    rng = np.random.default_rng(head_dim + 3 * heads)
    length = [1, 2, 15, 16, 17, 33, 127, 128, 129, 300, 517]
    new = [1] * len(length)
    pool, table, start, q = make(rng, cache, dtype, heads, group, head_dim, page, length, new)
    check_attention(dev, stream, pool, table, start, length, q, dtype, group)


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("heads,group,head_dim,page", [(2, 4, 128, 16), (1, 8, 64, 32),
                                                       (2, 1, 96, 64), (1, 5, 256, 16)])
def test_chunks(dev, stream, dtype, cache, heads, group, head_dim, page):
    """Chunks of many lengths, with and without positions before them, beside steps and idle
    sequences; more rows than the sequences have; strided Q."""
    rng = np.random.default_rng(head_dim + group)
    length = [1, 3, 70, 40, 9, 65, 200, 131, 0, 64]
    new = [1, 3, 70, 2, 0, 33, 17, 100, 0, 1]
    pool, table, start, q = make(rng, cache, dtype, heads, group, head_dim, page, length, new,
                                 gap=32, extra=5)
    check_attention(dev, stream, pool, table, start, length, q, dtype, group,
                    q_stride=heads * group * head_dim + 40)


@pytest.mark.parametrize("dtype,cache", [(D.BF16, D.BF16), (D.F16, D.E4M3), (D.F16, D.F16)])
@pytest.mark.parametrize("group", [1, 4])
def test_long_chunk(dev, stream, dtype, cache, group):
    """Several row tiles of one sequence, the last of odd size, behind and without a cached part."""
    rng = np.random.default_rng(group)
    length, new = [700, 333], [300, 333]
    pool, table, start, q = make(rng, cache, dtype, 1, group, 128, 32, length, new)
    check_attention(dev, stream, pool, table, start, length, q, dtype, group)


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_peaked(dev, stream, dtype, cache):
    """Scores of tens: one position holds the mass, the maximum moves late and often."""
    rng = np.random.default_rng(11)
    length, new = [400, 37, 260], [1, 5, 40]
    pool, table, start, q = make(rng, cache, dtype, 2, 4, 128, 16, length, new, q_std=6.0)
    check_attention(dev, stream, pool, table, start, length, q, dtype, 4)


@pytest.mark.parametrize("cache", [D.E4M3, D.I8])
@pytest.mark.parametrize("dtype,peak", [(D.F16, 1e-6), (D.F16, 3e3), (D.BF16, 1e-27),
                                        (D.BF16, 1e-6), (D.BF16, 1e20), (D.BF16, 3e28),
                                        (D.BF16, 1e35)])
def test_scales_far_from_one(dev, stream, cache, dtype, peak):
    """Scales whose products with probabilities leave f16's range, and f32's with the largest taken
    out: V alone is scaled (K keeps scores of order one), at random by the position."""
    rng = np.random.default_rng(12)
    length, new = [300, 50], [1, 20]
    pool, table, start, q = make(rng, cache, dtype, 1, 4, 64, 16, length, new)
    grow = np.float32(peak) * np.exp2(rng.uniform(-6, 3, pool.scale[1].shape)).astype(np.float32)
    pool.scale[1] = pool.scale[1] * grow
    got = run_attention(dev, stream, pool, table, start, length, q, dtype, 4)
    for b, n in enumerate(length):
        rows = slice(start[b], start[b + 1])
        kv = [pool.read(i, table[b], n) for i in range(2)]
        o, mean, reach = pg.attention(pg.widen(q[rows], dtype).astype(np.float64), kv,
                                      pool.there(table[b], n), new[b], n, 4)
        e = (64 + 8) * 2.0 ** -23 * reach[..., None] + 2.0 ** -20 + 2.0 ** -24 * (n / 8 + 64)
        # probabilities times scales are multiples of 2^-24 of a power of two of at most the
        # largest scale; codes reach 448 (127); O's own step is absolute below 2^-14
        most = float(pool.scale[1][table[b][:-(-n // 16)]][~np.isnan(
            pool.scale[1][table[b][:-(-n // 16)]])].max())
        tol = ((2.0 ** -11 * mean + pg.HALF[dtype] * np.abs(o)) * 1.01 + 2 * e * mean
               + (2.0 ** -25 if dtype == D.F16 else 0) + n * 2.0 ** -24 * most * pg.MOST[cache])
        assert (np.abs(pg.widen(got[rows], dtype) - o) <= tol).all()


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_hidden_values_do_not_show(dev, stream, dtype, cache):
    """NaN and infinities in slots past the lengths, in the chunk's own later tokens, in spare
    pages: the same bits as with plain values there."""
    rng = np.random.default_rng(13)
    heads, group, hd, page = 2, 4, 128, 16
    length, new = [75, 140, 33], [9, 70, 1]
    pool, table, start, q = make(rng, cache, dtype, heads, group, hd, page, length, new)
    clean = check_attention(dev, stream, pool, table, start, length, q, dtype, group)
    # the last token of the first two sequences is NaN and infinite: earlier rows do not see it
    for b, bad in ((0, np.nan), (1, np.inf)):
        pos = length[b] - 1
        for i in range(2):
            x = np.full((heads, hd), bad, np.float32)
            pool.put(i, table[b, pos // page], pos % page, x)
    odd = run_attention(dev, stream, pool, table, start, length, q, dtype, group)
    for b in range(3):
        rows = slice(start[b], start[b + 1] - (b < 2))
        x, y = (pg.widen(z[rows], dtype).astype(np.float64) for z in (clean, odd))
        assert np.isfinite(y).all()
        # two evaluations, each within the bound of the exact one (of order u)
        assert np.abs(x - y).max() <= 4 * pg.HALF[dtype] * np.abs(x).max()
    for b in range(2):
        assert not np.isfinite(pg.widen(odd[start[b + 1] - 1], dtype)).any()


@pytest.mark.parametrize("dtype,cache", [(D.BF16, D.BF16), (D.F16, D.I8)])
def test_missing_pages_and_odd_lengths(dev, stream, dtype, cache):
    """Pages that are not there are hidden, rows that see nothing give zeros, lengths past the
    table and fewer positions than tokens."""
    rng = np.random.default_rng(14)
    pool = pg.Pool(rng, cache, 12, 16, 2, 64)
    table = np.array([[0, -1, 1, 12], [2, 3, 2**31 - 1, -7], [-1, -1, -1, -1], [4, 5, 6, 7],
                      [8, 9, 10, 11]], np.int32)
    for b in range(5):
        pool.fill(rng, table[b], 64)
    length, new = [60, 40, 50, 5, 1000], [3, 20, 2, 9, 4]
    start = np.concatenate([[0], np.cumsum(new)]).tolist()
    q = pg.narrow(rng.standard_normal((start[-1], 8, 64)), dtype)
    got = check_attention(dev, stream, pool, table, start, length, q, dtype, 4)
    assert not got[start[2]:start[3]].any() and not got[start[3]:start[3] + 4].any()
    # starts and lengths that hold anything
    length = [3, -2**31, 64, 2**31 - 1, -1]
    check_attention(dev, stream, pool, table, [5, 2, -9, 30, 7, 2**31 - 1], length, q, dtype, 4)


@pytest.mark.parametrize("dtype,cache", [(D.BF16, D.BF16), (D.BF16, D.E4M3)])
def test_shared_pages(dev, stream, dtype, cache):
    """Sequences with the same pages: each as if alone."""
    rng = np.random.default_rng(15)
    pool, table, _, _ = make(rng, cache, dtype, 2, 4, 128, 16, [200], [1])
    table = np.repeat(table, 4, axis=0)
    length, new = [200, 200, 150, 64], [1, 1, 5, 64]
    start = np.concatenate([[0], np.cumsum(new)]).tolist()
    q = pg.narrow(rng.standard_normal((start[-1], 8, 128)), dtype)
    got = check_attention(dev, stream, pool, table, start, length, q, dtype, 4)
    q[1] = q[0]
    got = check_attention(dev, stream, pool, table, start, length, q, dtype, 4)
    # the runs that the positions are dealt to differ: the same to a rounding
    assert np.abs(pg.widen(got[0], dtype) - pg.widen(got[1], dtype)).max() < 2.0 ** -6


@pytest.mark.parametrize("batch", [100, 333])
def test_many_sequences(dev, stream, batch):
    rng = np.random.default_rng(batch)
    length = rng.integers(0, 90, batch).tolist()
    new = [min(n, int(x)) for n, x in zip(length, rng.integers(0, 3, batch))]
    pool, table, start, q = make(rng, D.BF16, D.BF16, 1, 4, 64, 16, length, new)
    check_attention(dev, stream, pool, table, start, length, q, D.BF16, 4)


@pytest.mark.parametrize("batch", [64, 65, 140])
def test_many_chunks(dev, stream, batch):
    """Chunks of several row tiles in as many sequences as one look at the lengths takes, and in
    more; idle sequences between."""
    rng = np.random.default_rng(batch)
    length = rng.integers(0, 200, batch).tolist()
    new = [0 if b % 9 == 4 else min(n, int(x))
           for b, (n, x) in enumerate(zip(length, rng.integers(0, 200, batch)))]
    pool, table, start, q = make(rng, D.E4M3, D.F16, 1, 4, 64, 16, length, new)
    check_attention(dev, stream, pool, table, start, length, q, D.F16, 4)


@pytest.mark.parametrize("batch", [1, 3, 70])
def test_nobody_has_new_tokens(dev, stream, batch):
    """Rows that belong to no sequence, behind sequences of many positions and of none."""
    rng = np.random.default_rng(batch)
    length = [900] + [0, 17] * (batch // 2)
    length = (length + [5])[:batch]
    pool, table, start, q = make(rng, D.BF16, D.BF16, 1, 4, 64, 16, length, [0] * batch, extra=80)
    check_attention(dev, stream, pool, table, start, length, q, D.BF16, 4)


def test_long_step_is_the_same_twice(dev, stream):
    """One sequence over many runs: within the bound, the same bits each time, also on the
    stream's own scratch."""
    rng = np.random.default_rng(16)
    pool, table, start, q = make(rng, D.BF16, D.BF16, 1, 4, 64, 64, [9001], [1])
    a = check_attention(dev, stream, pool, table, start, [9001], q, D.BF16, 4)
    b = run_attention(dev, stream, pool, table, start, [9001], q, D.BF16, 4)
    c = run_attention(dev, stream, pool, table, start, [9001], q, D.BF16, 4, workspace=0)
    assert np.array_equal(a, b) and np.array_equal(a, c)


def test_pool_past_4_gib(dev, stream):
    """Pages whose byte offsets pass 32 bits, and elements that do."""
    if dev.mem_info().free < 40 << 30:
        pytest.skip("needs 40 GiB of free memory")
    rng = np.random.default_rng(17)
    heads, hd, page = 8, 128, 256
    num = (1 << 32) // (heads * hd * page) + 3            # 2^32 elements and three pages
    small = pg.Pool(rng, D.BF16, 3, page, heads, hd)
    table = np.array([[0, 2, 1]], np.int32)
    small.fill(rng, table[0], 600)
    q = pg.narrow(rng.standard_normal((2, 16, hd)), D.BF16)
    want = run_attention(dev, stream, small, table, [0, 2], [600], q, D.BF16, 2)
    size = heads * hd * page
    far = np.array([0, num // 2, num - 1])                # where the three pages go
    bufs = []
    for x in small.data:
        b = dev.alloc(num * size, D.BF16)
        for i, p in enumerate(far):
            src = pg.put(dev, stream, x[i * size:(i + 1) * size])
            th._lib.check(th.lib().th_memcpy_dtod_async(
                C.c_void_p(b.as_raw_ptr() + int(p) * size * 2), C.c_void_p(src.as_raw_ptr()),
                size * 2, stream.handle))
            stream.synchronize()
        bufs.append(b)
    pages = th.KvPages(bufs[0], bufs[1], num, page, heads, hd, D.BF16)
    seqs = pg.batch(dev, stream, far[table].astype(np.int32), [0, 2], [600], 2)
    room = th.attention_paged_workspace_size(pages, seqs, 16)
    o, ws = dev.alloc(q.size, D.BF16), dev.alloc(room // 4, D.F32)
    th.attention_paged(pg.put(dev, stream, q), pages, seqs, o, 16, D.BF16, 0, ws, room, stream)
    assert np.array_equal(o.copy_to_host(stream).reshape(q.shape), want)
    out = [dev.alloc(heads * 600 * hd, D.BF16) for _ in range(2)]
    th.kv_cache_read(pages, seqs, out[0], out[1], 600, D.BF16, stream)
    for i in range(2):
        assert np.array_equal(
            out[i].copy_to_host(stream),
            pg.narrow(small.read(i, table[0], 600).astype(np.float32), D.BF16).reshape(-1))
    for b in bufs:
        b.free()
