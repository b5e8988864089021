"""Refusals of the 4-bit cache and page calls that need no GPU, and the plain
implementations that the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest
import torch

import _kv4ref as R


def _ops():
    from metalbench_b200 import _lib, build, ops
    if not _lib.LIB_PATH.exists():
        build.build()
    return ops


def test_host_tensors_are_refused():
    ops = _ops()
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    cache = torch.zeros(2, 1, R.BLOB, dtype=torch.uint8)
    x = torch.zeros(1, 1, 1, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv4_append(x, x, cache, i32(1, 1), i32(1))
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv4_gather(cache, i32(1, 1), i32(1), 1, i32(1))
    with pytest.raises(ValueError, match="CUDA"):
        ops.attention_kv4(x, cache, i32(1, 1), i32(1))
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_pages_extend(i32(1, 1), i32(1), i32(2), i32(1))
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_pages_fork([], i32(1, 1), i32(1), i32(2), i32(1))
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_pages_compact([], i32(1, 1), i32(1), i32(2))


def test_device_zero_is_a_device(monkeypatch):
    """And not the current one."""
    ops, asked = _ops(), []
    from metalbench_b200.decoder import PagedKV4Cache
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    for name in ("zeros", "full"):
        real = getattr(torch, name)
        monkeypatch.setattr(torch, name, lambda *a, real=real, device=None, **k: asked.append(torch.device(device)) or real(*a, **k))
    ops.kv4_cache(1, 1, 0)
    PagedKV4Cache(1, 64, 1, device=0)
    assert asked and set(asked) == {torch.device("cuda", 0)}
    asked.clear()
    ops.kv4_cache(1, 1)
    assert asked == [torch.device("cuda", 3)]


@pytest.fixture(scope="module")
def lib():
    _ops()
    from metalbench_b200 import _lib
    return _lib.lib()


FAKE = 1 << 20  # an aligned address that is refused before anything reads it


@pytest.mark.parametrize("change, word", [
    (dict(Dh=64), "head_dim"), (dict(Hq=3, Hkv=2), "multiple of Hkv"), (dict(B=-1), "sizes"),
    (dict(q=None), "null"), (dict(q=FAKE + 8), "aligned"), (dict(ldq=132), "aligned"), (dict(num_pages=0), "sizes"),
    (dict(max_pages=1 << 25), "pages"), (dict(S=1 << 28), "rows"), (dict(most=257), "max_kv_len"), (dict(most=0), "max_kv_len"), (dict(ws=None), "workspace"), (dict(ws_bytes=16), "workspace"),
    (dict(S=-1), "sizes"),
])
def test_attention_arguments(lib, change, word):
    a = dict(q=FAKE, ldq=1024, cache=FAKE, num_pages=4, table=FAKE, max_pages=4, kv_len=FAKE, most=256, start=None, B=2, S=1,
             Hq=8, Hkv=8, Dh=128, scale=0.1, out=FAKE, ldo=1024, ws=FAKE, ws_bytes=1 << 30)
    a.update(change)
    rc = lib.mb_attention_kv4_bf16(*a.values(), None)
    assert rc == -1 and word in lib.mb_last_error().decode()


@pytest.mark.parametrize("change, word", [
    (dict(k=None), "null"), (dict(k=FAKE + 2), "aligned"), (dict(Hkv=0), "sizes"), (dict(k1=129), "strides"), (dict(v2=-4), "strides"),
    (dict(S=-1), "sizes"),
])
def test_append_arguments(lib, change, word):
    a = dict(k=FAKE, v=FAKE, k0=1024, k1=128, k2=128, v0=1024, v1=128, v2=128, cache=FAKE, num_pages=4, Hkv=1, table=FAKE,
             max_pages=4, start=FAKE, new=None, most=None, B=2, S=8)
    a.update(change)
    rc = lib.mb_kv4_append_bf16(*a.values(), None)
    assert rc == -1 and word in lib.mb_last_error().decode()


@pytest.mark.parametrize("change, word", [
    (dict(table=None), "null"), (dict(max_pages=0), "sizes"), (dict(ws=FAKE + 4), "aligned"), (dict(ws_bytes=8), "workspace"),
    (dict(pools=[FAKE + 8]), "aligned"), (dict(sizes=[24]), "multiple of 16"), (dict(pools=[None]), "pools"),
])
def test_page_arguments(lib, change, word):
    a = dict(pools=[FAKE], sizes=[64], table=FAKE, lens=FAKE, refs=FAKE, B=2, max_pages=4, P=16, parent=FAKE, status=FAKE,
             ws=FAKE, ws_bytes=1 << 20)
    a.update(change)
    pools, sizes = (C.c_void_p * 1)(*a["pools"]), (C.c_int64 * 1)(*a["sizes"])
    args = (a["table"], a["lens"], a["refs"], a["B"], a["max_pages"], a["P"], a["parent"], a["status"], a["ws"], a["ws_bytes"])
    assert lib.mb_kv_pages_fork(pools, sizes, 1, *args, None) == -1
    assert word in lib.mb_last_error().decode()


def test_empty_calls_launch_nothing(lib):
    assert lib.mb_kv4_append_bf16(None, None, 0, 0, 0, 0, 0, 0, None, 1, 1, None, 1, None, None, None, 0, 4, None) == 0
    assert lib.mb_kv4_gather_f32(None, 1, 1, None, 1, None, None, 2, 0, None, None, None) == 0
    assert lib.mb_attention_kv4_bf16(None, 0, None, 1, None, 1, None, 64, None, 0, 1, 8, 8, 128, 1.0, None, 0, None, 0, None) == 0
    assert lib.mb_attention_kv4_workspace_bytes(0, 1, 8, 8, 4) == 0
    assert lib.mb_kv4_page_bytes(8) == 8 * R.BLOB


def test_a_wide_table_does_not_ask_for_the_memory_of_expanded_pages(lib):
    most = max(lib.mb_attention_kv4_workspace_bytes(1, 512, 64, 8, n) for n in (1 << 17, 1 << 20, 1 << 24, 1 << 29))
    assert 0 < most <= 6 << 30


def test_one_sequence_of_too_many_rows_and_pages(lib):
    """A negative scale takes the form whose row tiles and pages are counted in 32 bits."""
    a = dict(q=FAKE, ldq=8192, cache=FAKE, num_pages=4, table=FAKE, max_pages=64, kv_len=FAKE, most=4096, start=None, B=3, S=1 << 22,
             Hq=64, Hkv=8, Dh=128, scale=-0.1, out=FAKE, ldo=8192, ws=FAKE, ws_bytes=1 << 40)
    rc = lib.mb_attention_kv4_bf16(*a.values(), None)
    assert rc == -1 and "too many pages" in lib.mb_last_error().decode()


def test_plain_quantiser_is_within_half_a_step():
    rng = np.random.default_rng(0)
    x = R.bf16_round(rng.standard_normal((64, 128)) * np.exp(rng.uniform(-20, 20, (64, 1))))
    u, s, m = R.quantise(x)
    # half a step, and 15 steps of the scale's own rounding (half of bf16's eps)
    assert (np.abs(m[:, None] + s[:, None] * u - x) <= s[:, None] * (0.5 + 16 * 2 ** -8)).all()
    blob = np.zeros(R.BLOB, dtype=np.uint8)
    for t in range(64):
        R.put_token(blob, t, x[t], x[63 - t])
    got = R.get_pages(blob[None])
    assert np.array_equal(got["k"][0][0], u) and np.array_equal(got["v"][0][0], u[::-1])
    assert np.array_equal(got["k"][1][0], s) and np.array_equal(got["v"][2][0], m[::-1])


def test_plain_pages_keep_their_rules():
    P = R.Pages(np.full((3, 4), -1, np.int32), np.zeros(3, np.int32), np.zeros(6, np.int32))
    assert P.extend([65, 0, 64]) == 0 and P.table[0, :2].tolist() == [0, 1] and P.table[2, 0] == 2
    assert P.extend([64 * 4, 0, 0]) == -1
    assert P.extend([128, 128, 0]) == 1 and P.lens.tolist() == [65, 0, 64]
    assert P.fork([0, 0, -1], []) == 0 and P.table[1, :2].tolist() == [0, 3] and P.refs.tolist() == [2, 1, 0, 1, 0, 0]
    live, remap = P.compact([])
    assert live == 3 and remap.tolist() == [0, 1, -1, 2, -1, -1] and P.table[1, :2].tolist() == [0, 2]
