"""The paged cache's operators together, as a server runs them: prompts and steps through a layer,
a drawn token fed back, the same in captured graphs and on two streams at once."""
from ctypes import c_void_p

import numpy as np
import pytest

import tilers_hip as th
from tests import paged as pg
from tests.test_gpu_paged import bound
from tests.test_gpu_sample import plain
from tests.test_gpu_scratch_capture import GLOBAL, record

pytestmark = pytest.mark.gpu
D = th.TileDtype
BF = D.BF16


def bits(x):
    return pg.narrow(x, BF)


def real(b, stream, shape):
    """A bf16 buffer's values."""
    n = int(np.prod(shape))
    return pg.widen(b.copy_to_host(stream)[:n].reshape(shape), BF).astype(np.float64)


def load(b, x, stream):
    """x into the front of a buffer, zeros behind it."""
    x = np.ascontiguousarray(x).reshape(-1).view(b.dtype.host_dtype)
    b.copy_from_host(np.concatenate([x, np.zeros(b.count - x.size, x.dtype)]), stream)


class Layer:
    """One attention layer with an embedding and a head, random weights."""

    def __init__(self, dev, stream, rng, heads=8, kv=2, hd=64, hidden=256, vocab=1009):
        self.dev, self.heads, self.kv, self.hd, self.hidden, self.vocab = (
            dev, heads, kv, hd, hidden, vocab)
        self.embed = rng.standard_normal((vocab, hidden)).astype(np.float32)

        def weight(rows, cols):
            return pg.put(dev, stream, bits(rng.standard_normal((rows, cols)) / np.sqrt(rows) * 1.5))
        self.wq, self.wk, self.wv = (weight(hidden, n * hd) for n in (heads, kv, kv))
        self.wo, self.head = weight(heads * hd, hidden), weight(hidden, vocab)

    def buffers(self, total):
        a = self.dev.alloc
        return dict(x=a(total * self.hidden, BF), n=a(total * self.hidden, BF),
                    q=a(total * self.heads * self.hd, BF), k=a(total * self.kv * self.hd, BF),
                    v=a(total * self.kv * self.hd, BF), o=a(total * self.heads * self.hd, BF),
                    y=a(total * self.hidden, BF), logits=a(total * self.vocab, D.F32),
                    tokens=a(total, D.F32), u=a(total, D.F32), temp=a(total, D.F32),
                    top_k=a(total, D.F32), top_p=a(total, D.F32))

    def serve(self, b, pool, seqs, total, stream, workspace=None, room=0):
        """The paged operators alone, on the q, k, v and logits that are there."""
        th.kv_cache_write(pool.pages, seqs, b["k"], b["v"], BF, 0, stream)
        th.attention_paged(b["q"], pool.pages, seqs, b["o"], self.heads, BF, 0, workspace, room,
                           stream)
        self.draw(b, total, stream)

    def draw(self, b, total, stream):
        th.sample(b["logits"], b["tokens"], total, self.vocab, D.F32, b["u"], b["temp"],
                  b["top_k"], b["top_p"], stream=stream)

    def run(self, b, pool, seqs, total, stream, workspace=None, room=0):
        """Every row's next token, from rows of x; K and V go into the cache on the way."""
        h, w = self.hidden, self.hd
        th.rms_norm(b["x"], b["n"], total, h, 1e-5, BF, stream)
        for to, m, n in (("q", self.wq, self.heads * w), ("k", self.wk, self.kv * w),
                         ("v", self.wv, self.kv * w)):
            th.matmul(b["n"], m, b[to], total, h, n, BF, BF, stream=stream)
        th.kv_cache_write(pool.pages, seqs, b["k"], b["v"], BF, 0, stream)
        th.attention_paged(b["q"], pool.pages, seqs, b["o"], self.heads, BF, 0, workspace, room,
                           stream)
        th.matmul(b["o"], self.wo, b["y"], total, self.heads * w, h, BF, BF, stream=stream)
        th.matmul(b["y"], self.head, b["logits"], total, h, self.vocab, BF, D.F32, stream=stream)
        self.draw(b, total, stream)

    def fill(self, rng, b, tokens, stream):
        n = len(tokens)
        limits = dict(u=rng.random(n), temp=rng.uniform(0.5, 1.3, n), top_p=rng.uniform(0.5, 1, n))
        load(b["x"], bits(self.embed[tokens]), stream)
        for name, x in limits.items():
            limits[name] = x.astype(np.float32)
            load(b[name], limits[name], stream)
        limits["top_k"] = rng.integers(1, 60, n).astype(np.int32)
        load(b["top_k"], limits["top_k"], stream)
        return limits

    def check(self, b, host, table, start, length, total, limits, stream):
        """Each operator against its plain form on the inputs that it had; the drawn tokens."""
        k, v = (pg.widen(b[x].copy_to_host(stream)[:total * self.kv * self.hd]
                         .reshape(total, self.kv, self.hd), BF) for x in "kv")
        q = real(b["q"], stream, (total, self.heads, self.hd))
        o = real(b["o"], stream, (total, self.heads, self.hd))
        logits = b["logits"].copy_to_host(stream)[:total * self.vocab].reshape(total, -1)
        tokens = b["tokens"].copy_to_host(stream).view(np.int32)[:total]
        for s, n in enumerate(length):
            new = start[s + 1] - start[s]
            for i in range(new):
                pos = n - new + i
                page, row = table[s][pos // host.page], pos % host.page
                host.put(0, page, row, k[start[s] + i])
                host.put(1, page, row, v[start[s] + i])
            if new == 0:
                continue
            rows = slice(start[s], start[s + 1])
            want, mean, reach = pg.attention(q[rows], [host.read(i, table[s], n) for i in range(2)],
                                             host.there(table[s], n), new, n,
                                             self.heads // self.kv)
            tol = bound(want, mean, reach, BF, self.hd, n, host.dtype in pg.MOST)
            assert (np.abs(o[rows] - want) <= tol).all(), (s, np.abs(o[rows] - want).max())
        for r in range(total):
            _, may = plain(logits[r].astype(np.float64), float(limits["u"][r]),
                           float(limits["temp"][r]), int(limits["top_k"][r]),
                           float(limits["top_p"][r]))
            assert tokens[r] in may, (r, tokens[r])
        return tokens


def same_cache(pool, host):
    """The device's pool is the host's, untouched positions too."""
    for got, want in zip(pool.codes(), host.data):
        assert np.array_equal(got.view(want.dtype), want)
    for got, want in zip(pool.scales(), host.scale):
        if want is not None:
            assert np.array_equal(got, want, equal_nan=True)


@pytest.mark.parametrize("cache", [D.BF16, D.E4M3, D.I8])
def test_prompts_and_steps(dev, stream, cache):
    """Three prompts at once, a fourth sequence idle; then steps in which the fourth's prompt joins
    and a sequence ends; every operator checked at each call."""
    rng = np.random.default_rng(21)
    layer = Layer(dev, stream, rng)
    host = pg.Pool(rng, cache, 24, 16, layer.kv, layer.hd)
    pool = pg.DevicePool(dev, stream, host)
    table = pg.tables(rng, host, [90, 40, 60, 70])
    length, last = [0, 0, 0, 0], [0] * 4
    b = layer.buffers(200)
    plan = [[61, 1, 33, 0], [1, 1, 1, 0], [1, 1, 1, 47], [1, 0, 1, 1], [1, 0, 1, 1]]
    for new in plan:
        start = np.concatenate([[0], np.cumsum(new)]).tolist()
        tokens = np.concatenate([rng.integers(0, layer.vocab, n) if n > 1 or length[s] == 0
                                 else [last[s]] * n for s, n in enumerate(new)]).astype(int)
        length = [x + n for x, n in zip(length, new)]
        total = start[-1]
        limits = layer.fill(rng, b, tokens, stream)
        seqs = pg.batch(dev, stream, table, start, length, total)
        layer.run(b, pool, seqs, total, stream)
        got = layer.check(b, host, table, start, length, total, limits, stream)
        for s, n in enumerate(new):
            if n:
                last[s] = int(got[start[s + 1] - 1])
    same_cache(pool, host)


@pytest.mark.parametrize("cache", [D.BF16, D.E4M3])
def test_read_feeds_contiguous_attention(dev, stream, cache):
    """The cache read back and decoded over as one block of positions, beside the paged form."""
    rng = np.random.default_rng(22)
    B, L, heads, kv, hd = 3, 333, 8, 2, 128
    host = pg.Pool(rng, cache, 70, 16, kv, hd)
    table = pg.tables(rng, host, [L] * B)
    for s in range(B):
        host.fill(rng, table[s], L)
    pool = pg.DevicePool(dev, stream, host)
    seqs = pg.batch(dev, stream, table, range(B + 1), [L] * B, B)
    q = bits(rng.standard_normal((B, heads, hd)))
    qd, k, v, o, paged = (pg.put(dev, stream, q), dev.alloc(B * kv * 400 * hd, BF),
                          dev.alloc(B * kv * 400 * hd, BF), dev.alloc(q.size, BF),
                          dev.alloc(q.size, BF))
    th.kv_cache_read(pool.pages, seqs, k, v, 400, BF, stream)
    th.attention_decode(qd, k, v, o, B, L, 400, hd, heads, kv, BF, stream=stream)
    th.attention_paged(qd, pool.pages, seqs, paged, heads, BF, stream=stream)
    got, beside = real(o, stream, q.shape), real(paged, stream, q.shape)
    for s in range(B):
        kvs = [host.read(i, table[s], L) for i in range(2)]
        want, mean, reach = pg.attention(pg.widen(q[s:s + 1], BF).astype(np.float64), kvs,
                                         host.there(table[s], L), 1, L, heads // kv)
        tol = bound(want, mean, reach, BF, hd, L, cache in pg.MOST)
        assert (np.abs(beside[s] - want) <= tol).all()
        # the values were rounded to bf16 on the way: K by half a step moves a score by at most
        # 2^-8 reach, a weight by twice that relative to the others; V by half a step itself
        more = 0 if cache == BF else (4 * 2.0 ** -8 * reach[..., None] + 2.0 ** -8) * mean
        assert (np.abs(got[s] - want) <= tol + more).all()


class Step:
    """A layer's single-token step of six sequences on its own pool, workspace and buffers."""
    B = 6

    def __init__(self, dev, stream, seed, cache=D.E4M3):
        self.rng = rng = np.random.default_rng(seed)
        self.dev, self.layer = dev, Layer(dev, stream, rng)
        self.host = pg.Pool(rng, cache, 140, 16, self.layer.kv, self.layer.hd)
        self.length = [1, 40, 129, 300, 256, 511]
        self.table = pg.tables(rng, self.host, [n + 40 for n in self.length])
        for s, n in enumerate(self.length):
            self.host.fill(rng, self.table[s], n - 1)
        self.pool = pg.DevicePool(dev, stream, self.host)
        self.b = self.layer.buffers(self.B)
        self.start = list(range(self.B + 1))
        self.seqs = th.KvBatch(pg.put(dev, stream, self.table),
                               pg.put(dev, stream, np.asarray(self.start, np.int32)),
                               dev.alloc(self.B, D.F32), self.B, self.table.shape[1], self.B)
        self.lens = self.seqs._held[2]
        self.room = th.attention_paged_workspace_size(self.pool.pages, self.seqs, self.layer.heads)
        assert self.room > 0
        self.ws = dev.alloc(self.room // 4 + 1, D.F32)

    def next(self, stream):
        """New inputs and lengths."""
        self.limits = self.layer.fill(self.rng, self.b, self.rng.integers(0, self.layer.vocab,
                                                                          self.B), stream)
        self.lens.copy_from_host(np.asarray(self.length, np.int32).view(np.float32), stream)

    def call(self, stream):
        self.layer.run(self.b, self.pool, self.seqs, self.B, stream, self.ws, self.room)

    def check(self, stream):
        got = self.layer.check(self.b, self.host, self.table, self.start, self.length, self.B,
                               self.limits, stream)
        self.length = [n + 1 for n in self.length]
        return got


def test_a_captured_step(dev, stream):
    """Recorded once and replayed with other lengths, tokens and limits, the program's own work on
    the same operators between the replays; bit for bit what the calls give themselves."""
    step, other = Step(dev, stream, 23), Step(dev, stream, 24)
    step.next(stream)
    step.call(stream)
    step.check(stream)
    graph, run = record(stream, GLOBAL, lambda: step.call(stream))
    hip = th.lib()
    for _ in range(5):
        step.next(stream)
        assert hip.hipGraphLaunch(run, c_void_p(stream.handle)) == 0
        step.check(stream)
        same_cache(step.pool, step.host)
        first = [step.b[x].copy_to_host(stream) for x in ("o", "tokens")]
        step.layer.serve(step.b, step.pool, step.seqs, step.B, stream, step.ws, step.room)
        for x, name in zip(first, ("o", "tokens")):
            assert np.array_equal(x.view(np.uint8), step.b[name].copy_to_host(stream).view(np.uint8))
        other.next(stream)
        other.call(stream)
        other.check(stream)
        stream.synchronize()
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0


def test_two_streams(dev, stream):
    """Steps on two streams at once, one of them a graph, each with its own workspace; and chunks on
    both with the streams' own scratch."""
    a, b = Step(dev, stream, 25), Step(dev, stream, 26, D.I8)
    two = dev.create_stream()
    a.next(stream)
    a.call(stream)
    a.check(stream)
    graph, run = record(stream, GLOBAL, lambda: a.call(stream))
    hip = th.lib()
    for _ in range(4):
        a.next(stream)
        b.next(two)
        stream.synchronize()
        two.synchronize()
        assert hip.hipGraphLaunch(run, c_void_p(stream.handle)) == 0
        b.call(two)
        a.check(stream)
        b.check(two)
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0
    rng = np.random.default_rng(27)
    jobs = []
    for s in (stream, two):
        host = pg.Pool(rng, BF, 70, 16, 2, 128)
        table = pg.tables(rng, host, [1000])
        host.fill(rng, table[0], 1000)
        pool = pg.DevicePool(dev, s, host)
        q = bits(rng.standard_normal((100, 8, 128)))
        jobs.append([s, pool, pg.batch(dev, s, table, [0, 100], [1000], 100),
                     pg.put(dev, s, q), [dev.alloc(q.size, BF) for _ in range(4)]])
    for s, pool, seqs, q, out in jobs:
        th.attention_paged(q, pool.pages, seqs, out[0], 8, BF, stream=s)
        s.synchronize()
    for i in (1, 2, 3):
        for s, pool, seqs, q, out in jobs:
            th.attention_paged(q, pool.pages, seqs, out[i], 8, BF, stream=s)
    for s, pool, seqs, q, out in jobs:
        want = out[0].copy_to_host(s)
        assert np.isfinite(pg.widen(want, BF)).all()
        for o in out[1:]:
            assert np.array_equal(o.copy_to_host(s), want)
    two.synchronize()


def test_capture_without_a_workspace(dev, stream):
    """Refused where the call is split, recorded where it is not; the capture lives on."""
    rng = np.random.default_rng(28)
    host = pg.Pool(rng, BF, 40, 16, 2, 64)
    table = pg.tables(rng, host, [500])
    host.fill(rng, table[0], 500)
    pool = pg.DevicePool(dev, stream, host)
    long = pg.batch(dev, stream, table, [0, 1], [500], 1)
    short = pg.batch(dev, stream, table[:, :2], [0, 1], [30], 1)
    assert th.attention_paged_workspace_size(pool.pages, short, 4) == 0
    q = pg.put(dev, stream, bits(rng.standard_normal((1, 4, 64))))
    o, want = dev.alloc(256, BF), dev.alloc(256, BF)
    th.attention_paged(q, pool.pages, short, want, 4, BF, stream=stream)

    def body():
        with pytest.raises(th.HalError) as e:
            th.attention_paged(q, pool.pages, long, o, 4, BF, stream=stream)
        assert e.value.kind == "MemoryError" and "captured" in str(e.value)
        th.attention_paged(q, pool.pages, short, o, 4, BF, stream=stream)
    graph, run = record(stream, GLOBAL, body)
    hip = th.lib()
    for _ in range(3):
        assert hip.hipGraphLaunch(run, c_void_p(stream.handle)) == 0
        assert np.array_equal(o.copy_to_host(stream), want.copy_to_host(stream))
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0


def test_captured_sampling_of_long_rows(dev, stream):
    """Rows that an eager call spreads over many workgroups: recorded, they take one each."""
    rng = np.random.default_rng(29)
    rows, vocab = 3, 100003
    x = bits(rng.standard_normal((rows, vocab)) * 3)
    logits, tokens, u = pg.put(dev, stream, x), dev.alloc(rows, D.F32), dev.alloc(rows, D.F32)
    u.copy_from_host(np.zeros(rows, np.float32), stream)
    th.sample(logits, tokens, rows, vocab, BF, u, stream=stream)
    graph, run = record(stream, GLOBAL,
                        lambda: th.sample(logits, tokens, rows, vocab, BF, u, stream=stream))
    wide = pg.widen(x, BF).astype(np.float64)
    hip = th.lib()
    for _ in range(4):
        draw = rng.random(rows).astype(np.float32)
        u.copy_from_host(draw, stream)
        for call in (lambda: hip.hipGraphLaunch(run, c_void_p(stream.handle)),
                     lambda: th.sample(logits, tokens, rows, vocab, BF, u, stream=stream)):
            call()
            got = tokens.copy_to_host(stream).view(np.int32)
            assert all(t in plain(w, float(d))[1] for t, w, d in zip(got, wide, draw))
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0
