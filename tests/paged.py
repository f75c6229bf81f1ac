"""Plain forms of the paged cache's operators in 64 bits, and a small pool of pages to run them on
(used by tests/test_gpu_paged.py, test_gpu_serving_step.py and test_paged_plain.py)."""
from __future__ import annotations

import numpy as np

import tilers_hip as th
from oracle import oracle as orc

D = th.TileDtype
ORC = {D.F32: orc.F32, D.F16: orc.F16, D.BF16: orc.BF16}
MOST = {D.E4M3: 448.0, D.I8: 127.0}
#: half a step of each type, relative to the value
HALF = {D.F32: 2.0 ** -24, D.F16: 2.0 ** -11, D.BF16: 2.0 ** -8}


def e4m3_values() -> np.ndarray:
    """The 256 codes' values: sign, 4 exponent bits of bias 7, 3 mantissa bits; 0x7f is NaN."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v[(c & 0x7f) == 0x7f] = np.nan
    return np.where(c & 0x80, -v, v)


E4M3 = e4m3_values()
_POSITIVE = E4M3[:127]   # rising


def to_e4m3(x: np.ndarray) -> np.ndarray:
    """Nearest codes of finite x of at most 448 (1 + 2^-6), ties to the even code."""
    a = np.abs(x.astype(np.float64))
    hi = np.clip(np.searchsorted(_POSITIVE, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = _POSITIVE[hi] - a, a - _POSITIVE[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return (code | np.where(np.signbit(x), 0x80, 0)).astype(np.uint8)


def values(code: np.ndarray, dtype: D) -> np.ndarray:
    """Codes or 16-bit patterns as f64."""
    if dtype == D.E4M3:
        return E4M3[code]
    if dtype == D.I8:
        return code.astype(np.float64)
    return orc.widen(code.reshape(-1), ORC[dtype]).reshape(code.shape).astype(np.float64)


def narrow(x: np.ndarray, dtype: D) -> np.ndarray:
    x = np.ascontiguousarray(x, np.float32)
    return x if dtype == D.F32 else orc.narrow(x.reshape(-1), ORC[dtype]).reshape(x.shape)


def widen(x: np.ndarray, dtype: D) -> np.ndarray:
    return x if dtype == D.F32 else orc.widen(x.reshape(-1), ORC[dtype]).reshape(x.shape)


def quantise(x: np.ndarray, dtype: D):
    """Codes and scales of f32 rows [..., head_dim]."""
    with np.errstate(all="ignore"):
        a = np.abs(x).max(axis=-1)          # (NaN where there is one)
        fine, some = a < np.inf, a >= np.float32(1e-30)
        inv = np.where(fine & some, np.float32(MOST[dtype]) / a, 0).astype(np.float32)
        scale = np.where(fine, np.where(some, a / np.float32(MOST[dtype]), 0), np.nan)
        y = np.where(inv[..., None] != 0, x * inv[..., None], 0).astype(np.float32)
    return (to_e4m3(y) if dtype == D.E4M3 else np.rint(y).astype(np.int8)), scale.astype(np.float32)


class Pool:
    """A pool of pages on the host: codes (or 16-bit patterns) and scales, all of it garbage."""

    def __init__(self, rng, dtype, num_pages, page, heads, head_dim, gap=0, garbage=None):
        self.dtype, self.num_pages, self.page, self.heads, self.head_dim = (
            dtype, num_pages, page, heads, head_dim)
        self.stride = heads * page * head_dim + gap
        n = num_pages * self.stride
        self.scale = [None, None]
        if dtype in MOST:
            self.data = [rng.integers(0, 256, n, dtype=np.uint8).view(dtype.host_dtype)
                         for _ in range(2)]
            self.scale = [np.full((num_pages, heads, page), np.nan, np.float32) for _ in range(2)]
        else:
            odd = np.array([np.nan, np.inf, -np.inf, 7e4], np.float32)
            self.data = [narrow(odd[rng.integers(0, 4, n)], dtype) for _ in range(2)]
        if garbage is not None:
            for x in self.data:
                x[:] = garbage


    def fill(self, rng, b_table, length, peak=1.0):
        """Values of N(0, peak) (any codes, with scales, in 8 bits) at positions [0, length)."""
        for pos in range(length):
            page, row = b_table[pos // self.page], pos % self.page
            if not 0 <= page < self.num_pages:
                continue
            for i in range(2):
                x = (rng.standard_normal((self.heads, self.head_dim)) * peak).astype(np.float32)
                self.put(i, page, row, x)

    def put(self, i, page, row, x):
        """f32 rows of every head at a position."""
        at = page * self.stride + (np.arange(self.heads)[:, None] * self.page + row) \
            * self.head_dim + np.arange(self.head_dim)
        if self.dtype in MOST:
            code, scale = quantise(x, self.dtype)
            self.data[i][at] = code
            self.scale[i][page, :, row] = scale
        else:
            self.data[i][at] = narrow(x, self.dtype)

    def read(self, i, table, length):
        """f64 values [heads][length][head_dim]; zeros where a page is missing."""
        out = np.zeros((self.heads, length, self.head_dim))
        for pos in range(length):
            k = pos // self.page
            page, row = table[k] if k < len(table) else -1, pos % self.page
            if not 0 <= page < self.num_pages:
                continue
            at = page * self.stride + (np.arange(self.heads)[:, None] * self.page + row) \
                * self.head_dim + np.arange(self.head_dim)
            x = values(self.data[i][at], self.dtype)
            if self.dtype in MOST:
                x = x * self.scale[i][page, :, row, None].astype(np.float64)
            out[:, pos] = x
        return out

    def there(self, table, length):
        """Which of the first `length` positions have a page."""
        k = np.arange(length) // self.page
        page = np.where(k < len(table), np.append(table, -1)[np.minimum(k, len(table))], -1)
        return (page >= 0) & (page < self.num_pages)


def put(dev, stream, x: np.ndarray):
    """A device buffer of any array's bytes."""
    x = np.ascontiguousarray(x)
    dtype = {1: D.I8, 2: D.BF16, 4: D.F32}[x.itemsize]
    b = dev.alloc(max(1, x.size), dtype)
    if x.size:
        b.copy_from_host(x.reshape(-1).view(dtype.host_dtype), stream)
    return b


class DevicePool:
    def __init__(self, dev, stream, pool: Pool):
        self.pool, self.stream = pool, stream
        self.data = [put(dev, stream, x) for x in pool.data]
        self.scale = [None if x is None else put(dev, stream, x) for x in pool.scale]
        dense = pool.heads * pool.page * pool.head_dim
        self.pages = th.KvPages(self.data[0], self.data[1], pool.num_pages, pool.page, pool.heads,
                                pool.head_dim, pool.dtype, self.scale[0], self.scale[1],
                                0 if pool.stride == dense else pool.stride)

    def codes(self):
        return [x.copy_to_host(self.stream).view(self.pool.dtype.host_dtype) for x in self.data]

    def scales(self):
        return [None if x is None else x.copy_to_host(self.stream).reshape(y.shape)
                for x, y in zip(self.scale, self.pool.scale)]


def batch(dev, stream, table, start, length, total_q):
    table = np.asarray(table, np.int32)
    return th.KvBatch(put(dev, stream, table), put(dev, stream, np.asarray(start, np.int32)),
                      put(dev, stream, np.asarray(length, np.int32)), len(length), table.shape[1],
                      total_q)


def tables(rng, pool, lengths, spare=0):
    """Pages in any order for each sequence, -1 behind its last."""
    need = [-(-n // pool.page) for n in lengths]
    order = rng.permutation(pool.num_pages)
    table = np.full((len(lengths), max(1, max(need) + spare)), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table


def attention(q, kv, there, n, length, group):
    """o and, for the bound, sum p |v| and the largest sum |q k| / sqrt(D) of each row, for the n
    last positions of `length`: q [n][heads][D] in f64, kv two [kv_heads][held][D]."""
    k, v = kv
    held, d = k.shape[1], k.shape[2]
    o, mean, reach = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:2])
    for i in range(n):
        see = min(max(length - n + i + 1, 0), held)
        on = there[:see]
        if not on.any():
            continue
        for h in range(q.shape[1]):
            kk, vv = k[h // group, :see][on], v[h // group, :see][on]
            s = kk @ q[i, h] / np.sqrt(d)
            p = np.exp(s - s.max())
            p /= p.sum()
            o[i, h], mean[i, h] = p @ vv, p @ np.abs(vv)
            reach[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max() / np.sqrt(d)
    return o, mean, reach
