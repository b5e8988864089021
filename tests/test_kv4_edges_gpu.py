"""The 4-bit cache where its forms replace a number by another one: zeros and
constants among the values, weights rounded to fp16, wide tables, a status that
outlives its call. Against the plain 64-bit implementations (_kv4ref)."""
import numpy as np
import pytest
import torch

import _kv4ref as R
from test_kv4_gpu import bf, clean_status, i32, make_cache, make_table, ops, status  # noqa: F401

pytestmark = pytest.mark.gpu


def held(ops, k, v, table, P):
    """A cache of P pages with the tokens k, v [B, L, H, 128], as numpy."""
    cache = ops.kv4_cache(P, k.shape[2])
    ops.kv4_append(bf(k), bf(v), cache, i32(table), i32([0] * len(k)))
    return cache.cpu().numpy()


def attend(ops, q, cache, table, lens, first=None):
    return ops.attention_kv4(bf(q), torch.from_numpy(cache).cuda(), i32(table), i32(lens),
                             start_pos=None if first is None else i32(first)).double().cpu().numpy()


def near(got, ref, slack):
    err, tol = np.abs(got - ref), slack + 2 ** -8 * (np.abs(ref) + slack)  # and the output's rounding to bf16
    return float((err - tol).max()) <= 0


# ---------------------------------------------------------------------------
# values of zero, and values that are all alike
# ---------------------------------------------------------------------------
def strong_zeros(rng, where, octaves, B, L, Hkv, size, value=0.0):
    """Keys and values of N(0, 1) and size * N(0, 1); the tokens `where` have all
    dims of the value alike and scores about `octaves` above the others' mean, for
    q of mean 1: a key of b in all its dims scores 128 b / sqrt(128) log2(e) = 16.3 b octaves."""
    k, v = rng.standard_normal((B, L, Hkv, 128)), size * rng.standard_normal((B, L, Hkv, 128))
    k[:, where], v[:, where] = octaves / 16.3, value
    return R.bf16_round(k), R.bf16_round(v)


PAGE0 = list(range(64))
SOME = [0, 5, 63, 64, 130, 300, 511]
MOST = list(range(0, 500))


@pytest.mark.parametrize("size", [1.0, 0.1, 1e-3, 1e-6])
@pytest.mark.parametrize("octaves", [0, 6, 12])
@pytest.mark.parametrize("where", [PAGE0, SOME, MOST], ids=["page", "some", "most"])
def test_prompts_over_zero_values(ops, where, octaves, size):
    """Zeros count in the denominator and nowhere else: they must not take the
    bits of the values that stand beside them."""
    rng = np.random.default_rng(len(where) + octaves)
    B, S, Hq, Hkv, lens = 2, 512, 4, 2, np.array([700, 600])
    k, v = strong_zeros(rng, where, octaves, B, 700, Hkv, size)
    table, P = make_table(rng, [700, 700])
    cache = held(ops, k, v, table, P)
    q = R.bf16_round(rng.standard_normal((B, S, Hq, 128)) + 1)
    ref, _ = R.attention(q, cache, table, lens, lens - S)
    assert near(attend(ops, q, cache, table, lens, lens - S), ref, R.prompt_slack(q, cache, table, lens, lens - S))
    assert status() == 0


@pytest.mark.parametrize("size", [1.0, 0.1, 1e-3, 1e-6, 1e-10])
@pytest.mark.parametrize("octaves", [0, 6, 12])
@pytest.mark.parametrize("where", [PAGE0, SOME, MOST], ids=["page", "some", "most"])
@pytest.mark.parametrize("B, S", [(1, 1), (2, 1), (2, 4)])
def test_rows_over_zero_values(ops, B, S, where, octaves, size):
    rng = np.random.default_rng(len(where) + octaves)
    Hq, Hkv, lens = 8, 2, np.array([700, 600])[:B]
    k, v = strong_zeros(rng, where, octaves, B, 700, Hkv, size)
    table, P = make_table(rng, [700] * B)
    cache = held(ops, k, v, table, P)
    q = R.bf16_round(rng.standard_normal((B, S, Hq, 128)) + 1)
    ref, slack = R.attention(q, cache, table, lens, lens - S)
    assert near(attend(ops, q, cache, table, lens, lens - S), ref, slack)
    assert status() == 0


@pytest.mark.parametrize("value", [2.0 ** -20, -0.375, 1e4])
@pytest.mark.parametrize("octaves", [0, 8])
@pytest.mark.parametrize("S, Hq", [(1, 8), (4, 8), (512, 4)])
def test_constants_among_other_values(ops, S, Hq, octaves, value):
    """All dims of some values alike (scale 0, codes 0, a minimum of its own)."""
    rng = np.random.default_rng(octaves)
    Hkv, lens = 2, np.array([700, 600])
    k, v = strong_zeros(rng, SOME, octaves, 2, 700, Hkv, 0.5, value)
    table, P = make_table(rng, [700, 700])
    cache = held(ops, k, v, table, P)
    q = R.bf16_round(rng.standard_normal((2, S, Hq, 128)) + 1)
    ref, slack = R.attention(q, cache, table, lens, lens - S)
    slack = R.prompt_slack(q, cache, table, lens, lens - S) if S >= 512 else slack
    assert near(attend(ops, q, cache, table, lens, lens - S), ref, slack)


def test_scales_of_zero_beside_scales_of_every_size(ops):
    """Scales 2^-40 to 2^2 and, among them, scales of 0 with codes 0 and minima
    of 0, of the neighbours' size and far below it."""
    rng = np.random.default_rng(13)
    table, P = make_table(rng, [300])
    cache = make_cache(rng, P, 1)
    s = np.exp2(rng.integers(-40, 3, (P, 1, 64)).astype(np.float64))
    low = -7 * s
    for p in range(P):
        flat = rng.permutation(64)[:12]
        s[p, 0, flat] = 0
        low[p, 0, flat[4:8]] = 0
        low[p, 0, flat[8:]] = 2.0 ** -30
        codes = cache[p, 0, 4096: 8192].reshape(64, 64)
        codes[flat] = 0
    cache[..., 8448:] = np.stack([R.bf16_bits(s), R.bf16_bits(low)], -1).reshape(P, 1, 128).view(np.uint8)
    for S in (1, 3):
        q = R.bf16_round(rng.standard_normal((1, S, 8, 128)) * 4)
        ref, slack = R.attention(q, cache, table, [300], None)
        assert near(attend(ops, q, cache, table, [300]), ref, slack)


@pytest.mark.parametrize("S, Hq", [(1, 8), (4, 8), (512, 4)])
@pytest.mark.parametrize("exp", [-50, 60])
def test_zeros_beside_very_small_and_very_large_values(ops, S, Hq, exp):
    rng = np.random.default_rng(exp + 100)
    lens = np.array([700, 600])
    for where in (PAGE0, SOME, MOST):
        k, v = strong_zeros(rng, where, 3, 2, 700, 2, 2.0 ** exp)
        table, P = make_table(rng, [700, 700])
        cache = held(ops, k, v, table, P)
        q = R.bf16_round(rng.standard_normal((2, S, Hq, 128)) + 1)
        ref, slack = R.attention(q, cache, table, lens, lens - S)
        slack = R.prompt_slack(q, cache, table, lens, lens - S) if S >= 512 else slack
        assert near(attend(ops, q, cache, table, lens, lens - S), ref, slack)


# ---------------------------------------------------------------------------
# rounded weights
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("B, S, Hq, Hkv, L", [(1, 1, 8, 2, 700), (3, 1, 32, 8, 900), (2, 4, 8, 2, 300), (1, 1, 64, 8, 9000)])
def test_equal_values_come_back_whatever_their_weights(ops, B, S, Hq, Hkv, L):
    """Every token has the same value, so that the output is that value for any
    weights: a weight's own rounding must go the same way in the numerator's
    two parts (codes and minimum) and in the denominator. What may be off: n/16
    accumulations of 2^-23 and n/32 of 2^-24 of scale * code + |minimum|, the
    division and the reciprocal of the scale (2^-20 together), and weights
    under 2^-22 of the largest, which fp16 holds to 2^-33 of that."""
    rng = np.random.default_rng(L)
    x = np.tile(np.arange(16) - 7.0, 8)  # scale 1, minimum -7: exact, many of them 0
    lens = np.full(B, L)
    table, P = make_table(rng, lens)
    k = R.bf16_round(rng.standard_normal((B, L, Hkv, 128)))
    cache = held(ops, k, np.broadcast_to(x, k.shape).copy(), table, P)
    q = R.bf16_round(rng.standard_normal((B, S, Hq, 128)))
    got = attend(ops, q, cache, table, lens)
    size = x + 14  # scale * code + |minimum|
    tol = size * (L / 16 * 2 ** -23 + L / 32 * 2 ** -24 + 2 ** -20 + L * 2 ** -33)
    assert (np.abs(got - x) <= tol + 2 ** -8 * (np.abs(x) + tol)).all(), float(np.abs(got - x).max())


def test_a_long_share_has_no_bias(ops):
    """About 100 pages a warp of equal values, the minimum -7 and codes of 7: what the
    matrix unit cuts off of 16 products and its accumulator (less than 2^-24 of it
    each) may bias a page's four sums, 4 * 17 * 2^-24 of the codes' part in all, but
    not add up over the pages; sums with rounding have no mean error. (Sequences name
    the same few pages over and over.)"""
    rng = np.random.default_rng(8)
    B, Hq, P, M = 64, 8, 50, 2800
    x = np.tile(np.arange(16) - 7.0, 8)
    k = R.bf16_round(rng.standard_normal((1, P * 64, 1, 128)))
    cache = held(ops, k, np.broadcast_to(x, k.shape).copy(), np.arange(P, dtype=np.int32)[None], P)
    q = R.bf16_round(rng.standard_normal((B, 1, Hq, 128)))
    for n in (8, 3):  # query rows a sequence: one column tile, two
        rows = q if n == 8 else np.repeat(q, 3, 1)
        got = attend(ops, rows, cache, rng.integers(0, P, (B, M)).astype(np.int32), np.full(B, M * 64))
        bias = got[..., x == 0].mean() / 7
        print("bias", bias)
        assert abs(bias) <= 4 * 17 * 2 ** -24, bias


# ---------------------------------------------------------------------------
# wide tables and bounds
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("scale", [128 ** -0.5, -(128 ** -0.5)])
def test_many_sequences_under_a_wide_table(ops, scale):
    """512 x 64 rows of 8 heads, 65536 columns: 2^30 pages of row tiles at the
    table's width, far fewer in use. The expanded form (scale > 0) plans without
    that list, the other one takes fewer sequences at a time."""
    rng = np.random.default_rng(5)
    B, S, Hq, M = 512, 64, 8, 65536
    lens = np.zeros(B, dtype=np.int64)
    lens[[0, 300, 510, 511]] = 130, 64, 1, 200
    small, P = make_table(rng, lens)
    table = torch.full((B, M), -1, dtype=torch.int32, device="cuda")
    table[:, : small.shape[1]] = i32(small)
    cache = make_cache(rng, P, 1)
    c = torch.from_numpy(cache).cuda()
    q = torch.randn(B, S, Hq, 128, device="cuda").to(torch.bfloat16)
    got = ops.attention_kv4(q, c, table, i32(lens), start_pos=i32(lens - S), scale=scale)
    for b in range(B):
        if not lens[b]:
            continue
        # scale * q = |scale| * (+-q), exactly: the slack's term for a score's error is a multiple of the scale
        # that it is given, and means its magnitude
        x = np.sign(scale) * q[b: b + 1].double().cpu().numpy()
        at = (cache, small[b: b + 1], lens[b: b + 1], lens[b: b + 1] - S, abs(scale))
        ref, slack = R.attention(x, *at)
        assert near(got[b: b + 1].double().cpu().numpy(), ref, np.maximum(slack, R.prompt_slack(x, *at)))
    assert (got[torch.from_numpy(lens == 0).cuda()] == 0).all() and status() == 0


@pytest.mark.parametrize("S", [1, 3, 80])
@pytest.mark.parametrize("most", [None, 130, 1000])
def test_every_bound_gives_the_defined_rows(ops, S, most):
    rng = np.random.default_rng(18)
    table = np.arange(300, dtype=np.int32).reshape(2, 150)
    cache = make_cache(rng, 300, 2)
    q, n = R.bf16_round(rng.standard_normal((2, S, 8, 128))), [130, 100]
    got = ops.attention_kv4(bf(q), torch.from_numpy(cache).cuda(), i32(table), i32(n), max_kv_len=most).double().cpu().numpy()
    ref, slack = R.attention(q, cache, table, n, None)
    assert near(got, ref, np.maximum(slack, R.prompt_slack(q, cache, table, n, None)))


# ---------------------------------------------------------------------------
# numbers at the end of the range
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("S", [7, 70])
def test_a_range_that_overflows_reads_back_as_nan(ops, S):
    """max - min is an fp32 number: from 2^128 on the token has no scale. Just
    below, its largest code still stands for a finite number."""
    big = 3.3895313892515355e38  # the largest bf16
    x = np.zeros((1, S, 1, 128))
    x[0, :, 0] = np.linspace(-1, 1, 128)
    x[0, 1, 0, :2] = -big, big
    x[0, 3, 0] = np.linspace(-big / 2, big / 2, 128)
    x[0, 5, 0, :2] = -2.0 ** 126, big  # the range rounds to 2^128 and more
    x = R.bf16_round(x)
    cache = ops.kv4_cache(2, 1)
    ops.kv4_append(bf(x), bf(-x), cache, i32([[0, 1]]), i32([0]))
    for got, y in zip(ops.kv4_gather(cache, i32([[0, 1]]), i32([0]), S, i32([S])), (x, -x)):
        got = got.cpu().numpy()[0, :, 0]
        for s in range(S):
            if s in (1, 5):
                assert np.isnan(got[s]).all()
            else:
                u, sc, m = R.quantise(y[0, s, 0])
                want = (m + sc * u).astype(np.float32)
                assert np.isfinite(want).all() and np.array_equal(got[s], want)


# ---------------------------------------------------------------------------
# one caller's mistake
# ---------------------------------------------------------------------------
def test_a_bad_page_stays_its_callers(ops):
    """The mark that a table entry out of range leaves is there until it is
    cleared; other kernels of the device go on."""
    from metalbench_b200 import harness
    ops.attention_kv4(torch.zeros(1, 1, 1, 128, dtype=torch.bfloat16, device="cuda"), ops.kv4_cache(1, 1), i32([[7]]), i32([5]))
    assert status() == 8
    name = next(n for n in sorted(harness.registry_all()) if "transpose" in n)
    assert harness.evaluate(name, warmup=1, iters=2, ref_warmup=0, ref_iters=1)["correct"]
    assert status() == 8


# ---------------------------------------------------------------------------
# pools of other types and sizes
# ---------------------------------------------------------------------------
def test_pages_of_the_bf16_cache_and_of_real_size(ops):
    """Forks and a compaction of bf16 key and value pages [pages, heads, 64, 128],
    of 68 KiB 4-bit pages (five pieces of the copy) and of 8.5 KiB ones together."""
    rng = np.random.default_rng(31)
    B, M, P = 5, 6, 30
    ref = R.Pages(np.full((B, M), -1, np.int32), np.zeros(B, np.int32), np.zeros(P, np.int32))
    pools = [torch.randn(P, 2, 64, 128, device="cuda").to(torch.bfloat16), torch.randn(P, 3, 64, 128, device="cuda").to(torch.bfloat16),
             torch.randint(0, 256, (P, 8, R.BLOB), dtype=torch.uint8, device="cuda"),
             torch.randint(0, 256, (P, 1, R.BLOB), dtype=torch.uint8, device="cuda")]
    data = [p.view(torch.uint8).cpu().numpy().copy() for p in pools]
    table, lens, refs = i32(ref.table), i32(ref.lens), i32(ref.refs)

    def same():
        for a, b in ((table, ref.table), (lens, ref.lens), (refs, ref.refs), *zip((p.view(torch.uint8) for p in pools), data)):
            assert np.array_equal(a.cpu().numpy(), b)

    new = [300, 130, 64, 7, 0]
    assert int(ops.kv_pages_extend(table, lens, refs, i32(new))[1]) == ref.extend(new) == 0
    for parent in ([0, 0, 1, 3, 0], [1, 1, -1, 0, 4], [-1, 1, 1, 3, 3], [0, -1, 2, 3, 3]):
        assert int(ops.kv_pages_fork(pools, table, lens, refs, i32(parent))) == ref.fork(parent, data) == 0
        same()
        live, remap = ref.compact(data)
        got, n = ops.kv_pages_compact(pools, table, lens, refs)
        assert int(n) == live and np.array_equal(got.cpu().numpy(), remap)
        same()


def test_pools_that_overlap_are_refused(ops):
    """A page moved in one would be another page of the other."""
    both = torch.zeros(5, 64, dtype=torch.uint8, device="cuda")
    t, n, r = i32([[0, 1]]), i32([70]), i32([1, 1, 0, 0])
    for pools in ([both[:4], both[1:]], [both[1:], both[:4]]):
        with pytest.raises(ValueError, match="pool"):
            ops.kv_pages_fork(pools, t, n, r, i32([0]))
        with pytest.raises(ValueError, match="pool"):
            ops.kv_pages_compact(pools, t, n, r)
    halves = torch.zeros(8, 64, dtype=torch.uint8, device="cuda")
    assert int(ops.kv_pages_fork([halves[:4], halves[4:]], t, n, r, i32([0]))) == 0


# ---------------------------------------------------------------------------
# the decoder layer's lengths
# ---------------------------------------------------------------------------
def test_lengths_that_are_no_int32_of_the_device_are_refused(ops):
    """Their addresses go to the kernels as they are."""
    from metalbench_b200.decoder import PagedKV4Cache, PagedKVCache
    from test_decoder_gpu import _layer, _weights
    rng = np.random.default_rng(3)
    layer = _layer(torch, _weights(rng, 512, 4, 2, 512), 512, 4, 2, 512, 10000.0)
    x = bf(rng.standard_normal((2, 1, 512)))
    pairs = i32([[0, 9], [1, 9]])
    for cache in (PagedKV4Cache(2, 64, 2).layer(0), PagedKVCache(2, 64, 2)):
        for bad in (torch.tensor([1, 1]), torch.tensor([1, 1], dtype=torch.int32), i32([1, 1]).long(), i32([1]), i32([1, 1, 1]), pairs[:, 0]):
            with pytest.raises(ValueError, match="kv_len"):
                layer(x, cache, i32([0, 0]), kv_len=bad, max_kv_len=64)
            with pytest.raises(ValueError, match="start_pos"):
                layer(x, cache, bad, max_kv_len=64)
    with pytest.raises(ValueError, match="new_len"):
        layer(x, PagedKV4Cache(2, 64, 2).layer(0), i32([0, 0]), new_len=pairs[:, 1])


# ---------------------------------------------------------------------------
# the cache's status
# ---------------------------------------------------------------------------
def test_the_status_keeps_what_a_replayed_step_lacked(ops):
    """Two pages, 64 tokens a step: the third replay finds none, whatever ran between."""
    from metalbench_b200.decoder import PagedKV4Cache
    cache = PagedKV4Cache(1, 256, 1, num_pages=2)
    full, none = i32([64]), i32([0])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        cache.extend(none)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.extend(full)
        cache.fork(none)  # a second operation of the step, served
    for length, lacking in ((64, 0), (128, 0), (128, 1), (128, 1)):
        g.replay()
        cache.extend(none)
        cache.compact()
        assert cache.seq_len.tolist() == [length] and int(cache.status) == lacking
    cache.clear_status()
    cache.extend(none)
    assert int(cache.status) == 0
    cache.block_table[0, 1] = 9
    cache.compact()
    cache.extend(none)
    assert int(cache.status) == -1
    g.replay()
    assert int(cache.status) == -1


def test_filling_a_cache_that_is_too_small_is_an_error(ops):
    from metalbench_b200.decoder import DecoderConfig
    from metalbench_b200.stack import DecoderStack
    from test_decoder_gpu import _weights
    rng = np.random.default_rng(3)
    W = [[bf(w) for w in _weights(rng, 512, 4, 2, 512)]]
    st = DecoderStack(DecoderConfig(512, 4, 2, 512), 1, 3, 256, weights=W, kv_bits=4, num_pages=5)
    with pytest.raises(ValueError, match="lacks 1"):
        st.fill_cache_random(100)
    assert st.kv4.seq_len.tolist() == [0, 0, 0]
    st.fill_cache_random(64)
    assert st.kv4.seq_len.tolist() == [64] * 3
    with pytest.raises(ValueError, match="longer"):
        st.fill_cache_random(50)
    st.close()
