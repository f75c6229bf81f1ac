"""The plain forms that the paged cache's GPU tests measure against, checked on the CPU."""
import numpy as np
import pytest
import torch

import tilers_hip as th
from tests import paged as pg

D = th.TileDtype


def test_eight_bit_values():
    code = np.arange(256, dtype=np.uint8)
    want = torch.from_numpy(code).view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(pg.E4M3, want.astype(np.float64), equal_nan=True)


def test_eight_bit_rounding():
    rng = np.random.default_rng(1)
    mid = (pg._POSITIVE[1:] + pg._POSITIVE[:-1]) / 2          # ties
    x = np.concatenate([mid, -mid, rng.standard_normal(4000) * 100, rng.standard_normal(4000) * 0.01,
                        [0.0, -0.0, 448.0, -448.0]]).astype(np.float32)
    x = x[np.abs(x) <= 448]
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(pg.to_e4m3(x), want)


@pytest.mark.parametrize("dtype", [D.E4M3, D.I8])
def test_quantise(dtype):
    """Values come back to half a step, the largest exactly to a rounding; rows of zeros, tiny ones
    and what is no number."""
    rng = np.random.default_rng(2)
    x = (rng.standard_normal((50, 64)) * 10.0 ** rng.integers(-20, 20, (50, 1))).astype(np.float32)
    code, scale = pg.quantise(x, dtype)
    back = pg.values(code, dtype) * scale[:, None].astype(np.float64)
    top = np.abs(x).max(1, keepdims=True).astype(np.float64)
    step = 2.0 ** -4 * np.abs(x) + top / 448 * 2.0 ** -10 if dtype == D.E4M3 else top / 254
    assert (np.abs(back - x) <= step * (1 + 2.0 ** -18) + top * 2.0 ** -22).all()
    odd = np.zeros((4, 16), np.float32)
    odd[1] = 1e-31
    odd[2, 3], odd[3, 5] = np.inf, np.nan
    code, scale = pg.quantise(odd, dtype)
    assert (pg.values(code, dtype) == 0).all()
    assert scale[0] == 0 and scale[1] == 0 and np.isnan(scale[2:]).all()


def test_pool_round_trip():
    rng = np.random.default_rng(3)
    pool = pg.Pool(rng, D.BF16, 5, 16, 2, 32, gap=16)
    table = pg.tables(rng, pool, [37, 20])
    assert sorted(table[table >= 0]) == sorted(set(table[table >= 0]))
    x = pg.widen(pg.narrow(rng.standard_normal((2, 32)), D.BF16), D.BF16)
    pool.put(1, table[0][2], 4, x)
    assert np.array_equal(pool.read(1, table[0], 37)[:, 36], x)
    table[0, 1] = 99
    assert (pool.read(1, table[0], 37)[:, 16:32] == 0).all()
    assert np.array_equal(pool.there(table[0], 60), np.isin(np.arange(60) // 16, [0, 2]))


def test_attention():
    """The mask by position and the missing pages, against the whole softmax."""
    rng = np.random.default_rng(4)
    n, length, held = 4, 9, 9
    q = rng.standard_normal((n, 6, 16))
    kv = [rng.standard_normal((2, held, 16)) for _ in range(2)]
    there = np.ones(held, bool)
    there[2:4] = False
    o, mean, reach = pg.attention(q, kv, there, n, length, 3)
    for i in range(n):
        on = there & (np.arange(held) <= length - n + i)
        for h in range(6):
            s = torch.from_numpy(np.where(on, kv[0][h // 3] @ q[i, h] / 4, -np.inf))
            p = torch.softmax(s, 0).numpy()
            assert np.allclose(o[i, h], p @ kv[1][h // 3], rtol=1e-12, atol=1e-14)
            assert (mean[i, h] >= np.abs(o[i, h]) - 1e-12).all()
            assert reach[i, h] >= np.abs(s.numpy()[on]).max()
    o, _, _ = pg.attention(q, kv, np.zeros(held, bool), n, length, 3)
    assert (o == 0).all()
