"""What the paged cache's entry points refuse, and their index arithmetic: no GPU needed."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

import tilers_hip as th
from tilers_hip import _build, _lib

ROOT = Path(__file__).resolve().parents[1]
D = th.TileDtype
OK = dict(num_pages=4, page_size=16, num_kv_heads=2, head_dim=64, dtype=D.BF16, k=1 << 20,
          v=1 << 20, k_scale=None, v_scale=None, page_stride=0, page_table=4, q_start=4, kv_len=4,
          batch=2, max_pages=3, total_q=5)


def structs(**change):
    a = {**OK, **change}
    pages = th.KvPages(a["k"], a["v"], a["num_pages"], a["page_size"], a["num_kv_heads"],
                       a["head_dim"], a["dtype"], a["k_scale"], a["v_scale"], a["page_stride"])
    seqs = th.KvBatch(a["page_table"], a["q_start"], a["kv_len"], a["batch"], a["max_pages"],
                      a["total_q"])
    return pages, seqs


def test_index_arithmetic(tmp_path):
    exe = tmp_path / "paged_index"
    cmd = ["g++", "-O1", "-g", "-std=c++17", "-Wall", "-Wextra", "-fsanitize=address,undefined",
           "-fno-sanitize-recover=all", "-I", str(_build.CSRC),
           str(ROOT / "tests" / "native" / "paged_index_host.cpp"), "-o", str(exe)]
    out = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert out.returncode == 0, out.stdout
    out = subprocess.run([str(exe)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True,
                         timeout=60)
    assert out.returncode == 0, out.stdout


CALLS = {
    "write": lambda p, s: th.kv_cache_write(p, s, 1 << 20, 1 << 20, D.BF16),
    "read": lambda p, s: th.kv_cache_read(p, s, 1 << 20, 1 << 20, 48, D.BF16),
    "attention": lambda p, s: th.attention_paged(1 << 20, p, s, 1 << 20, 4, D.BF16),
}


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("change,says", [
    (dict(dtype=D.F32), "dtype must be"),
    (dict(num_kv_heads=0), "num_kv_heads == 0"),
    (dict(num_kv_heads=0xffffffff), "2^32 elements"),
    (dict(head_dim=0), "head_dim"), (dict(head_dim=24), "head_dim"),
    (dict(head_dim=272), "head_dim"),
    (dict(page_size=0), "page_size"), (dict(page_size=8), "page_size"),
    (dict(page_size=48), "page_size"), (dict(page_size=1 << 17), "page_size"),
    (dict(num_pages=0), "num_pages"), (dict(num_pages=1 << 31), "num_pages"),
    (dict(page_stride=2047), "page_stride"), (dict(page_stride=2056), "page_stride"),
    (dict(page_stride=1 << 62), "page_stride"),
    (dict(k=0), "null pages"), (dict(v=0), "null pages"), (dict(k=(1 << 20) + 8), "aligned"),
    (dict(dtype=D.E4M3), "k_scale"), (dict(dtype=D.I8, k_scale=16), "v_scale"),
    (dict(dtype=D.I8, k_scale=16, v_scale=20), "aligned"),
    (dict(batch=0x7fffffff), "below 2^31"), (dict(total_q=1 << 31), "below 2^31"),
    (dict(kv_len=0), "null page_table"), (dict(page_table=0), "null page_table"),
    (dict(kv_len=6), "4-byte"),
])
def test_refusals(call, change, says):
    with pytest.raises(th.HalError) as e:
        CALLS[call](*structs(**change))
    assert e.value.kind == "KernelError" and says in str(e.value)


def test_refusals_of_one_call():
    def refused(says, f, kind="KernelError"):
        with pytest.raises(th.HalError) as e:
            f()
        assert says in str(e.value) and e.value.kind == kind

    p, s = structs()
    a = 1 << 20
    refused("unknown dtype", lambda: th.kv_cache_write(p, s, a, a, D.E4M3))
    refused("stride", lambda: th.kv_cache_write(p, s, a, a, D.BF16, stride=127))
    refused("stride", lambda: th.kv_cache_write(p, s, a, a, D.BF16, stride=132))
    refused("stride", lambda: th.kv_cache_write(p, s, a, a, D.F32, stride=130))
    refused("stride is too large", lambda: th.kv_cache_write(p, s, a, a, D.F32, stride=1 << 60))
    many = structs(total_q=1 << 28)[1]
    refused("grid too large", lambda: th.kv_cache_write(p, many, a, a, D.F32))
    refused("grid too large", lambda: th.kv_cache_read(p, s, a, a, 0x7fffffff, D.F32))
    refused("grid too large", lambda: th.attention_paged(a, p, structs(batch=1 << 28,
                                                                       total_q=1 << 29)[1], a, 2,
                                                         D.BF16))
    refused("null pointer", lambda: th.kv_cache_write(p, s, 0, a, D.BF16))
    refused("aligned", lambda: th.kv_cache_write(p, s, a, a + 2, D.BF16))
    refused("unknown dtype", lambda: th.kv_cache_read(p, s, a, a, 8, D.I8))
    refused("null pointer", lambda: th.kv_cache_read(p, s, a, 0, 8, D.F32))
    refused("aligned", lambda: th.kv_cache_read(p, s, a + 8, a, 8, D.F32))
    refused("below 2^31", lambda: th.kv_cache_read(p, s, a, a, 1 << 31, D.F32))
    refused("F16 or BF16", lambda: th.attention_paged(a, p, s, a, 4, D.F32))
    refused("dtype of Q", lambda: th.attention_paged(a, p, s, a, 4, D.F16))
    refused("num_heads", lambda: th.attention_paged(a, p, s, a, 0, D.BF16))
    refused("num_heads", lambda: th.attention_paged(a, p, s, a, 5, D.BF16))
    refused("q_stride", lambda: th.attention_paged(a, p, s, a, 4, D.BF16, q_stride=255))
    refused("q_stride", lambda: th.attention_paged(a, p, s, a, 4, D.BF16, q_stride=260))
    refused("q_stride is too large",
            lambda: th.attention_paged(a, p, s, a, 4, D.BF16, q_stride=1 << 60))
    refused("null pointer", lambda: th.attention_paged(0, p, s, a, 4, D.BF16))
    refused("aligned", lambda: th.attention_paged(a, p, s, a + 8, 4, D.BF16))
    big, many = structs(total_q=1 << 30)
    refused("total_q * num_heads", lambda: th.attention_paged(a, big, many, a, 4, D.BF16))
    assert th.attention_paged_workspace_size(p, s, 4) == 0   # 48 positions: nothing is split
    p, s = structs(max_pages=30)
    room = th.attention_paged_workspace_size(p, s, 4)
    assert room > 0
    refused("workspace", lambda: th.attention_paged(a, p, s, a, 4, D.BF16, workspace=a,
                                                    workspace_bytes=room - 1), "MemoryError")
    refused("workspace must be", lambda: th.attention_paged(
        a, p, s, a, 4, D.BF16, workspace=a + 4, workspace_bytes=room))
    null = _lib.KvPagesStruct(), _lib.KvBatchStruct()
    f = th.lib().th_kv_cache_read
    assert f(None, C.byref(null[1]), a, a, 8, 0, None) == _lib.TH_KERNEL_ERROR
    assert f(p._ref, None, a, a, 8, 0, None) == _lib.TH_KERNEL_ERROR
    assert th.lib().th_attention_paged_workspace_size(None, None, 4) == 0
    assert th.attention_paged_workspace_size(p, s, 5) == 0


def test_nothing_to_do_is_no_error():
    """(No GPU here: any launch would fail.)"""
    for change in (dict(batch=0, kv_len=0, q_start=0, page_table=0), dict(total_q=0)):
        p, s = structs(**change)
        th.kv_cache_write(p, s, 0, 0, D.BF16)
        th.attention_paged(0, p, s, 0, 4, D.BF16)
        assert th.attention_paged_workspace_size(p, s, 4) == 0
    p, s = structs(batch=0)
    th.kv_cache_read(p, s, 0, 0, 9, D.F32)
    p, s = structs()
    th.kv_cache_read(p, s, 0, 0, 0, D.F32)


def test_sample_refusals():
    a = 1 << 20

    def refused(says, *args, **kw):
        with pytest.raises(th.HalError) as e:
            th.sample(*args, **kw)
        assert says in str(e.value) and e.value.kind == "KernelError"

    refused("unknown dtype", a, a, 2, 10, D.I8, a)
    refused("stride is less", a, a, 2, 10, D.F32, a, stride=9)
    refused("stride is too large", a, a, 2, 10, D.F32, a, stride=1 << 60)
    refused("vocab == 0", a, a, 2, 0, D.F32, a)
    refused("at most 2^23", a, a, 2, (1 << 23) + 1, D.F32, a)
    refused("at most 2^23", a, a, 2, 1 << 31, D.F32, a)
    refused("below 2^31", a, a, 1 << 31, 2, D.F32, a)
    refused("grid too large", a, a, 1 << 22, 2, D.F32, a)
    for i in range(3):
        p = [a, a, a]
        p[i] = 0
        refused("null pointer", p[0], p[1], 2, 10, D.F32, p[2])
    refused("aligned", a + 2, a, 2, 10, D.F32, a)
    refused("aligned", a + 1, a, 2, 10, D.BF16, a)
    for name in ("temperature", "top_k", "top_p", "min_p"):
        refused("aligned", a, a, 2, 10, D.BF16, a, **{name: a + 2})
    th.sample(0, 0, 0, 10, D.F32, 0)   # no rows


def test_eight_bit_types_elsewhere_are_refused():
    a = 1 << 20
    with pytest.raises(th.HalError):
        th.softmax(a, a, 2, 2, D.E4M3)
    with pytest.raises(th.HalError):
        th.matmul(a, a, a, 2, 2, 2, D.I8, D.F32)
    assert D.E4M3.itemsize == D.I8.itemsize == 1
    assert D.E4M3.host_dtype == np.uint8 and D.I8.host_dtype == np.int8
