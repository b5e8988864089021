"""The 4-bit paged cache, the attention over it and the page operations on the
GPU against plain 64-bit implementations (_kv4ref)."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import _kv4ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from metalbench_b200 import ops as o
    o.init(0)
    return o


@pytest.fixture(autouse=True)
def clean_status(ops):
    from metalbench_b200 import _lib
    _lib.call("mb_clear_device_status")
    yield
    _lib.call("mb_clear_device_status")


def status():
    from metalbench_b200 import _lib
    v = C.c_uint32(0)
    _lib.call("mb_device_status", C.byref(v))
    return v.value


def i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).cuda()


def bf(x):
    return torch.from_numpy(np.asarray(x, dtype=np.float32)).to(torch.bfloat16).cuda()


def make_cache(rng, num_pages, H, strong=True):
    """A filled cache (uint8 numpy) with codes, scales and minima as they come."""
    c = rng.integers(0, 256, (num_pages, H, R.BLOB), dtype=np.uint8)
    scale = np.exp(rng.normal(-1.2, 0.5 if strong else 0.0, (num_pages, H, 128)))
    low = -7.5 * scale + rng.normal(0, 0.2, scale.shape)
    par = np.stack([R.bf16_bits(scale), R.bf16_bits(low)], -1).astype(np.uint16)
    c[..., 8192:] = par.reshape(num_pages, H, 256).view(np.uint8)
    return c


def make_table(rng, lens, extra=2, width=None):
    counts = [R.pages_of(int(n)) for n in lens]
    P = sum(counts) + extra
    M = width or max(1, max(counts))
    t = np.full((len(lens), M), -1, np.int32)
    order = rng.permutation(P)
    at = 0
    for b, n in enumerate(counts):
        t[b, :n] = order[at: at + n]
        at += n
    return t, P


# ---------------------------------------------------------------------------
# storing and reading back
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("B, S, H, starts, new", [
    (1, 1, 1, [0], None), (3, 1, 8, [63, 64, 200], None), (2, 70, 2, [0, 33], [70, 5]),
    (4, 5, 3, [1, 60, 127, 0], [0, 5, 1, 3]), (1, 257, 4, [129], None),
])
@pytest.mark.parametrize("strided", [False, True])
def test_append_writes_exactly_the_defined_bytes(ops, B, S, H, starts, new, strided):
    rng = np.random.default_rng(S * 10 + H)
    ends = [s + (S if new is None else n) for s, n in zip(starts, new or [S] * B)]
    table, P = make_table(rng, ends)
    cache = rng.integers(0, 256, (P, H, R.BLOB), dtype=np.uint8)
    k, v = (R.bf16_round(rng.standard_normal((B, S, H, 128)) * np.exp(rng.uniform(-3, 3, (B, S, H, 1)))) for _ in range(2))
    want = cache.copy()
    for b in range(B):
        for s in range(S if new is None else new[b]):
            pos = starts[b] + s
            for h in range(H):
                R.put_token(want[table[b, pos // 64], h], pos % 64, k[b, s, h], v[b, s, h])
    c = torch.from_numpy(cache).cuda()
    if strided:  # rows of a fused projection
        row = torch.zeros(B, S, 3 * H, 128, dtype=torch.bfloat16, device="cuda")
        row[:, :, :H], row[:, :, 2 * H:] = bf(k), bf(v)
        kt, vt = row[:, :, :H], row[:, :, 2 * H:]
    else:
        kt, vt = bf(k), bf(v)
    ops.kv4_append(kt, vt, c, i32(table), i32(starts), None if new is None else i32(new))
    assert np.array_equal(c.cpu().numpy(), want)
    kb, vb = ops.kv4_gather(c, i32(table), i32(starts), S, i32(ends))
    for got, x in ((kb, k), (vb, v)):
        u, s, m = R.quantise(x)
        ref = (m[..., None] + s[..., None] * u).astype(np.float32)  # one rounding
        for b in range(B):
            ref[b, ends[b] - starts[b]:] = 0
        assert np.array_equal(got.cpu().numpy(), ref)
    assert status() == 0


def test_append_of_odd_rows(ops):
    """All dims alike, NaN, infinities, subnormals, the type's extremes: each
    only ever changes its own token."""
    big = 3.3895313892515355e38  # the largest bf16
    edge = np.linspace(-19, 11, 128)  # scale 2: a number next to nothing lies next to the border 9.5
    edge[3:6] = -3.67e-7, 3.67e-7, 0
    rows = [edge, np.arange(128) / 8 - 4, np.full(128, 1.5), np.zeros(128), np.linspace(-1, 1, 128), np.full(128, np.nan), np.full(128, np.inf),
            np.full(128, 1e-39), np.linspace(0, 9e-39, 128), np.linspace(-1e4, 1e4, 128), np.linspace(0, big, 128)]
    x = np.stack([R.bf16_round(r) for r in rows])[None, :, None]
    x[0, 4, 0, 5] = np.nan
    cache = ops.kv4_cache(1, 1)
    S = x.shape[1]
    ops.kv4_append(bf(x), bf(x[:, ::-1].copy()), cache, i32([[0]]), i32([0]))
    k, v = (t.cpu().numpy()[0, :, 0] for t in ops.kv4_gather(cache, i32([[0]]), i32([0]), S, i32([S])))
    for i in range(S):
        y = bf(x[0, i, 0]).double().cpu().numpy()
        if not np.isfinite(y).all():
            assert np.isnan(k[i]).all() and np.isnan(v[S - 1 - i]).all(), i
        else:
            u, s, m = R.quantise(y)
            ref = (m + s * u).astype(np.float32)
            assert np.array_equal(k[i], ref) and np.array_equal(v[S - 1 - i], ref), i


@pytest.mark.parametrize("S", [5, 64, 200])
def test_append_next_to_a_border(ops, S):
    """Quotients next to halves, from numbers far smaller than the range: the
    difference to the minimum is not a number of 32 bits. Both storing forms."""
    rng = np.random.default_rng(S)
    x = np.empty((1, S, 2, 128))
    for i in range(S):
        for h in range(2):
            j = rng.integers(-14, 0)  # scale 2, the minimum an odd number: 0 is a border
            x[0, i, h] = rng.uniform(2 * j + 1, 2 * j + 31, 128)
            x[0, i, h, :2] = 2 * j + 1, 2 * j + 31
            x[0, i, h, 2:40] = rng.choice([-1, 0, 1], 38) * 2.0 ** rng.integers(-36, -14, 38)
            x[0, i, h] = rng.permutation(x[0, i, h]) * 2.0 ** rng.integers(-60, 60)
    x = R.bf16_round(x)
    cache = ops.kv4_cache(4, 2)
    ops.kv4_append(bf(x), bf(-x), cache, i32([[3, 1, 0, 2]]), i32([9]))
    for got, want in zip(ops.kv4_gather(cache, i32([[3, 1, 0, 2]]), i32([9]), S, i32([S + 9])), (x, -x)):
        u, s, m = R.quantise(want)
        assert np.array_equal(got.cpu().numpy(), (m[..., None] + s[..., None] * u).astype(np.float32))


def test_append_skips_bad_pages_and_positions(ops):
    rng = np.random.default_rng(3)
    cache = torch.from_numpy(rng.integers(0, 256, (3, 2, R.BLOB), dtype=np.uint8)).cuda()
    before = cache.clone()
    k = bf(rng.standard_normal((4, 2, 2, 128)))
    table = i32([[-1], [3], [2], [1]])
    ops.kv4_append(k, k, cache, table, i32([0, 5, 63, -1]))  # no page, beyond the pool, past the table, before it
    changed = (cache != before).any(-1).cpu().numpy()
    assert changed.tolist() == [[False, False], [True, True], [True, True]]  # slot 63 of page 2, slot 0 of page 1
    assert status() == 8
    kb, _ = ops.kv4_gather(cache, table, i32([0, 5, 0, 0]), 1, i32([1, 6, 64, 1]))
    assert (kb[:2] == 0).all() and torch.isfinite(kb[3]).all()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def check_attention(ops, rng, B, S, Hq, Hkv, lens, first=None, scale=None, amp=1.0, garbage=True):
    table, P = make_table(rng, np.maximum(lens, 0))
    cache = make_cache(rng, P, Hkv)
    if garbage:  # what stands past the end of a sequence may be anything
        for b, n in enumerate(lens):
            if n > 0 and n % 64:
                blob = cache[table[b, n // 64]]
                for par in (8192, 8448):
                    blob[:, par + 4 * (n % 64): par + 256] = rng.choice([0xFF, 0x7F, 0x80], blob[:, par + 4 * (n % 64): par + 256].shape)
    q = R.bf16_round(rng.standard_normal((B, S, Hq, 128)) * amp)
    got = ops.attention_kv4(bf(q), torch.from_numpy(cache).cuda(), i32(table), i32(lens),
                            start_pos=None if first is None else i32(first), scale=scale)
    ref, slack = R.attention(q, cache, table, lens, first, 128 ** -0.5 if scale is None else scale)
    err = np.abs(got.double().cpu().numpy() - ref)
    tol = slack + 2 ** -8 * (np.abs(ref) + slack)  # the output's own rounding to bf16
    assert (err <= tol).all(), float((err - tol).max())
    assert status() == 0


@pytest.mark.parametrize("Hq, Hkv", [(1, 1), (8, 8), (8, 1), (16, 1), (6, 2), (24, 8), (40, 8)])
@pytest.mark.parametrize("lens", [[1], [64, 65, 0], [63, 128, 700, 1, 0, 2000]])
def test_decode_heads_and_lengths(ops, Hq, Hkv, lens):
    check_attention(ops, np.random.default_rng(Hq * 100 + len(lens)), len(lens), 1, Hq, Hkv, lens)


@pytest.mark.parametrize("S", [2, 3, 5, 16, 33])
@pytest.mark.parametrize("Hq, Hkv", [(4, 4), (8, 2), (5, 1)])
def test_causal_rows(ops, S, Hq, Hkv):
    rng = np.random.default_rng(S)
    lens = np.array([S, S + 61, 300, 0, 1])
    check_attention(ops, rng, 5, S, Hq, Hkv, lens, first=lens - S)  # some rows stand before the first key


@pytest.mark.parametrize("S, Hq, Hkv, lens, causal", [
    (200, 3, 1, [190, 450, 0], True), (128, 2, 2, [128], True), (129, 4, 1, [129, 1000], False),
    (64, 8, 2, [200, 64, 0, 1], True), (65, 4, 4, [129, 65], False), (130, 5, 1, [130, 700], True),
    (257, 8, 8, [300], True), (64, 16, 2, [128, 500, 63], False),
])
def test_pieces_of_a_prompt(ops, S, Hq, Hkv, lens, causal):
    """Many rows a sequence: the cache is expanded to fp16 pages first."""
    rng = np.random.default_rng(S + Hq)
    lens = np.array(lens)
    table, P = make_table(rng, lens)
    cache = make_cache(rng, P, Hkv)
    for b, n in enumerate(lens):  # what stands past the end of a sequence may be anything
        if n % 64:
            cache[table[b, n // 64], :, 8192 + 4 * (n % 64): 8448] = 0xFF
            cache[table[b, n // 64], :, 8448 + 4 * (n % 64):] = 0xFF
    q = R.bf16_round(rng.standard_normal((len(lens), S, Hq, 128)))
    first = lens - S if causal else None  # some rows stand before the first key
    got = ops.attention_kv4(bf(q), torch.from_numpy(cache).cuda(), i32(table), i32(lens), start_pos=None if first is None else i32(first))
    # either form may be taken: unpacked pages round weights of codes (2^-11 of scale * code and of the minimum
    # apart, which may cancel in the sum), expanded ones the values themselves
    ref, slack = R.attention(q, cache, table, lens, first)
    slack = np.maximum(slack, R.prompt_slack(q, cache, table, lens, first))
    err = np.abs(got.double().cpu().numpy() - ref)
    tol = slack + 2 ** -8 * (np.abs(ref) + slack)
    assert (err <= tol).all(), float((err - tol).max())
    if causal:  # the last rows again, few at a time: the other form
        few = ops.attention_kv4(bf(q[:, -7:]), torch.from_numpy(cache).cuda(), i32(table), i32(lens), start_pos=i32(first + S - 7))
        err = np.abs(got[:, -7:].double().cpu().numpy() - few.double().cpu().numpy())
        assert (err <= tol[:, -7:] * 2).all()
    neg = ops.attention_kv4(bf(q[:, :, :]), torch.from_numpy(cache).cuda(), i32(table), i32(lens), scale=-128 ** -0.5)
    ref, slack = R.attention(q, cache, table, lens, None, -(128 ** -0.5))
    assert (np.abs(neg.double().cpu().numpy() - ref) <= np.abs(slack) + 2 ** -8 * (np.abs(ref) + np.abs(slack))).all()
    assert status() == 0


def scaled_params(cache, at, exps):
    """`cache` with the bf16 parameters at `at` times 2^exps[page, head]."""
    out = cache.copy()
    par = out[:, :, at: at + 256].copy().view(np.uint16)
    par = np.where(par & 0x7F80, (par.astype(np.int64) + (exps[:, :, None] << 7)).astype(np.uint16), 0)
    out[:, :, at: at + 256] = par.astype(np.uint16).view(np.uint8)
    return out


@pytest.mark.parametrize("q_exp, k_exp, v_lo, v_hi", [
    (100, -100, 0, 1), (-100, 100, 0, 1), (0, 0, 100, 101), (0, 0, -100, -99), (0, 0, -12, 13), (0, 0, 24, 25), (0, 0, 12, 13), (30, -30, -40, 41),
])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("S, Hq", [(129, 4), (512, 8)])
def test_pieces_of_a_prompt_over_the_range_of_bf16(ops, S, Hq, q_exp, k_exp, v_lo, v_hi, causal):
    """Keys, values and rows far outside fp16's own range, values of one page far from another's."""
    rng = np.random.default_rng(7)
    Hkv, lens = 2, np.array([129, 400, 700])
    table, P = make_table(rng, lens)
    cache = make_cache(rng, P, Hkv)
    cache = scaled_params(cache, 8192, k_exp + rng.integers(-1, 2, (P, Hkv)))
    cache = scaled_params(cache, 8448, rng.integers(v_lo, v_hi, (P, Hkv)))
    q = R.bf16_round(rng.standard_normal((3, S, Hq, 128))) * 2.0 ** (q_exp + rng.integers(-1, 2, (3, S, Hq, 1)))
    first = lens - S if causal else None
    got = ops.attention_kv4(bf(q), torch.from_numpy(cache).cuda(), i32(table), i32(lens), start_pos=None if first is None else i32(first))
    # the form without expanded pages rounds weights of codes, so it errs by scale * code and minimum apart, not by
    # their sum alone; and it takes value scales below 2^-90 for that: 15 codes of it
    ref, slack = R.attention(q, cache, table, lens, first)
    slack = R.prompt_slack(q, cache, table, lens, first) if S >= 512 else slack + 15 * 2.0 ** -90
    err = np.abs(got.double().cpu().numpy() - ref)
    tol = slack + 2 ** -8 * (np.abs(ref) + slack)
    assert (err <= tol).all(), float((err - tol).max())
    assert status() == 0


@pytest.mark.parametrize("S, Hq, B, L", [(128, 4, 1, 3000), (100, 3, 2, 1500), (300, 8, 1, 2049)])
@pytest.mark.parametrize("causal", [False, True])
def test_few_row_tiles_over_many_keys(ops, S, Hq, B, L, causal):
    """The keys of a row tile are cut among several CTAs and joined."""
    rng = np.random.default_rng(S)
    lens = np.array([L, L // 2 + 3][:B])
    table, P = make_table(rng, lens)
    cache = make_cache(rng, P, 1)
    q = R.bf16_round(rng.standard_normal((B, S, Hq, 128)))
    first = np.array([L - S, -S // 2][:B]) if causal else None  # the second one: rows that see nothing, few keys seen
    got = ops.attention_kv4(bf(q), torch.from_numpy(cache).cuda(), i32(table), i32(lens), start_pos=None if first is None else i32(first))
    ref, slack = R.attention(q, cache, table, lens, first)
    slack = np.maximum(slack, R.prompt_slack(q, cache, table, lens, first))
    err = np.abs(got.double().cpu().numpy() - ref)
    tol = slack + 2 ** -8 * (np.abs(ref) + slack)
    assert (err <= tol).all(), float((err - tol).max())
    assert status() == 0


def test_prompts_on_two_streams_and_in_a_graph(ops):
    """Both at once, each with its own workspace; then captured and replayed with other inputs."""
    rng = np.random.default_rng(3)
    sets = []
    for S, L in ((300, 2000), (130, 3500)):
        table, P = make_table(rng, np.array([L, L // 2]))
        q = bf(rng.standard_normal((2, S, 8, 128)))
        args = [q, torch.from_numpy(make_cache(rng, P, 2)).cuda(), i32(table), i32([L, L // 2]), i32([L - S, 0])]
        sets.append((args, ops.attention_kv4(*args)))
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for st, (args, _) in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(ops.attention_kv4(*args))
        torch.cuda.synchronize()
        assert all(torch.equal(g, want) for g, (_, want) in zip(got, sets))
    graphs, outs = [], []
    for args, _ in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.attention_kv4(*args))
        graphs.append(g)
    for args, _ in sets:
        args[0].mul_(-1)
        args[3].sub_(40)
    want = [ops.attention_kv4(*args) for args, _ in sets]
    for g in graphs + graphs:
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want)) and status() == 0


@pytest.mark.parametrize("S, Hq, Hkv, lens, causal", [
    (512, 8, 2, [129, 400, 700], True), (512, 8, 2, [129, 400, 700], False), (128, 8, 2, [5000], True), (1, 32, 8, [3000, 7, 900], True),
])
def test_the_same_call_gives_the_same_bits(ops, S, Hq, Hkv, lens, causal):
    rng = np.random.default_rng(S)
    lens = np.array(lens)
    table, P = make_table(rng, lens)
    cache = torch.from_numpy(make_cache(rng, P, Hkv)).cuda()
    q = bf(rng.standard_normal((len(lens), S, Hq, 128)))
    start = i32(lens - S) if causal else None
    want = ops.attention_kv4(q, cache, i32(table), i32(lens), start_pos=start)
    for _ in range(40):
        assert torch.equal(ops.attention_kv4(q, cache, i32(table), i32(lens), start_pos=start), want)


@pytest.mark.parametrize("at", ["k", "v"])
@pytest.mark.parametrize("S, Hq, Hkv, L", [(4, 8, 1, 300), (33, 4, 2, 400), (512, 8, 2, 700), (128, 4, 1, 3000)])
def test_only_rows_that_see_a_nan_become_one(ops, S, Hq, Hkv, L, at):
    """A key or value that is no number, behind some rows' positions."""
    rng = np.random.default_rng(L)
    lens, first = np.array([L, L]), np.array([L - S, L - S])
    table, P = make_table(rng, lens)
    cache = make_cache(rng, P, Hkv)
    q = R.bf16_round(rng.standard_normal((2, S, Hq, 128)))
    ref, slack = R.attention(q, cache, table, lens, first)
    slack = np.maximum(slack, R.prompt_slack(q, cache, table, lens, first))
    hide = S // 2  # rows from here see the position
    pos = L - S + hide
    bad = cache.copy()
    bad[table[0, pos // 64], 0, (8192 if at == "k" else 8448) + 4 * (pos % 64):][:4] = 0xFF  # scale and minimum: NaN
    got = ops.attention_kv4(bf(q), torch.from_numpy(bad).cuda(), i32(table), i32(lens), start_pos=i32(first)).double().cpu().numpy()
    G = Hq // Hkv
    assert np.isnan(got[0, hide:, :G]).all()
    got[0, hide:, :G] = ref[0, hide:, :G]
    assert (np.abs(got - ref) <= slack + 2 ** -8 * (np.abs(ref) + slack)).all()
    assert status() == 0


@pytest.mark.parametrize("B, S, Hq, Hkv", [(1, 4, 8, 2), (3, 4, 8, 2), (2, 2, 16, 1), (2, 70, 4, 4), (2, 400, 8, 2)])
@pytest.mark.parametrize("what", [float("inf"), float("nan"), 3e38, 1e20])
def test_padding_rows_may_hold_anything(ops, B, S, Hq, Hkv, what):
    """Rows behind a sequence's new tokens share tiles with its own."""
    rng = np.random.default_rng(S)
    lens = np.array([S + 70, S + 200, S][:B])
    table, P = make_table(rng, lens)
    cache = make_cache(rng, P, Hkv)
    first = lens - S
    q = R.bf16_round(rng.standard_normal((B, S, Hq, 128)))
    ref, slack = R.attention(q, cache, table, lens, first)
    slack = np.maximum(slack, R.prompt_slack(q, cache, table, lens, first))
    keep = S // 2
    q[:, keep:] = what
    got = ops.attention_kv4(bf(q), torch.from_numpy(cache).cuda(), i32(table), i32(lens), start_pos=i32(first))
    err = np.abs(got.double().cpu().numpy() - ref)[:, :keep]
    assert (err <= (slack + 2 ** -8 * (np.abs(ref) + slack))[:, :keep]).all(), float(err.max())
    assert status() == 0


@pytest.mark.parametrize("B, S, Hq, Hkv, L", [(1, 1, 8, 2, 700), (3, 1, 32, 8, 3000), (2, 5, 8, 2, 500), (2, 300, 8, 2, 600)])
def test_the_output_may_take_the_place_of_the_queries(ops, B, S, Hq, Hkv, L):
    rng = np.random.default_rng(L)
    lens = np.array([L, L // 2, 0][:B])
    table, P = make_table(rng, lens)
    cache = torch.from_numpy(make_cache(rng, P, Hkv)).cuda()
    q = bf(R.bf16_round(rng.standard_normal((B, S, Hq, 128))))
    want = ops.attention_kv4(q, cache, i32(table), i32(lens))
    for _ in range(3):
        both = q.clone()
        ops.attention_kv4(both, cache, i32(table), i32(lens), out=both)
        assert torch.equal(both, want)


@pytest.mark.parametrize("S", [1, 4, 70])
def test_rows_that_see_nothing_are_zero(ops, S):
    rng = np.random.default_rng(9)
    if S < 64:
        check_attention(ops, rng, 3, S, 8, 2, np.array([100, 100, 64]), first=np.array([-100, -2, -(2 ** 31)]))
    cache, table = torch.from_numpy(make_cache(rng, 6, 2)).cuda(), i32([[0, 1], [2, 3], [4, 5]])
    q = bf(rng.standard_normal((3, S, 8, 128)))
    got = ops.attention_kv4(q, cache, table, i32([100, 0, 64]), start_pos=i32([-S, 5, -(2 ** 31)]))
    assert (got == 0).all()


def test_start_far_past_the_end_sees_every_key(ops):
    check_attention(ops, np.random.default_rng(10), 2, 3, 8, 2, np.array([100, 64]), first=np.array([2 ** 31 - 1, 64]))
    rng = np.random.default_rng(10)
    cache, table = torch.from_numpy(make_cache(rng, 3, 2)).cuda(), i32([[0, 1], [2, 2]])
    q = bf(rng.standard_normal((2, 80, 8, 128)))
    far, every = (ops.attention_kv4(q, cache, table, i32([100, 64]), start_pos=p) for p in (i32([2 ** 31 - 1, 64]), None))
    assert torch.equal(far, every)


def test_whole_cta_shares_and_many_units(ops):
    """More (sequence, head) units than shares, more sequences than one launch
    plans (512), and one unit over all shares."""
    rng = np.random.default_rng(11)
    lens = rng.integers(0, 80, 700)
    check_attention(ops, rng, 700, 1, 2, 2, lens, garbage=False)
    check_attention(ops, rng, 513, 3, 6, 1, np.minimum(lens[:513], 70), first=np.minimum(lens[:513], 70) - 3)
    check_attention(ops, rng, 70, 1, 16, 16, rng.integers(0, 200, 70), garbage=False)
    check_attention(ops, rng, 1, 1, 8, 1, np.array([70001]), garbage=False)


@pytest.mark.parametrize("Hq, Hkv, S, L, width", [
    (32, 8, 1, 517, 9), (8, 1, 1, 1, 1), (64, 8, 1, 20000, 400), (40, 8, 3, 777, 2000), (16, 16, 1, 4097, 65),
    (4, 2, 5, 130, 3), (8, 8, 1, 0, 4), (48, 24, 2, 3000, 47), (128, 64, 1, 130, 300), (16, 2, 40, 900, 15),
])
def test_one_sequence(ops, Hq, Hkv, S, L, width):
    """A single sequence: clusters of CTAs to a unit, of every size."""
    rng = np.random.default_rng(L)
    table, P = make_table(rng, [L], width=width)
    cache = make_cache(rng, P, Hkv)
    q = R.bf16_round(rng.standard_normal((1, S, Hq, 128)))
    got = ops.attention_kv4(bf(q), torch.from_numpy(cache).cuda(), i32(table), i32([L]), start_pos=i32([L - S]))
    ref, slack = R.attention(q, cache, table, [L], [L - S])
    err = np.abs(got.double().cpu().numpy() - ref)
    assert (err <= slack + 2 ** -8 * (np.abs(ref) + slack)).all()
    assert status() == 0


def test_large_scores_and_small_values(ops):
    rng = np.random.default_rng(12)
    check_attention(ops, rng, 2, 1, 8, 2, np.array([500, 64]), amp=30.0)
    check_attention(ops, rng, 2, 2, 8, 2, np.array([500, 64]), first=np.array([498, 62]), scale=1e-3)


def test_value_scales_of_very_different_size(ops):
    """Weights are rounded with their value scale in: a token with small values
    and nearly all of the weight is not lost beside large ones."""
    rng = np.random.default_rng(13)
    table, P = make_table(rng, [300])
    cache = make_cache(rng, P, 1)
    par = cache[..., 8448:].copy().view(np.uint16).reshape(P, 1, 64, 2)
    s = np.exp2(rng.integers(-40, 3, (P, 1, 64)).astype(np.float64))
    par[..., 0], par[..., 1] = R.bf16_bits(s), R.bf16_bits(-7 * s)
    s[0, 0, :5] = 0  # all dims alike: codes are zero
    cache[..., 8448:] = par.reshape(P, 1, 128).view(np.uint8).reshape(P, 1, 256)
    q = R.bf16_round(rng.standard_normal((1, 1, 8, 128)) * 4)
    got = ops.attention_kv4(bf(q), torch.from_numpy(cache).cuda(), i32(table), i32([300])).double().cpu().numpy()
    ref, slack = R.attention(q, cache, table, [300], None)
    assert (np.abs(got - ref) <= slack + 2 ** -8 * (np.abs(ref) + slack)).all()


def test_constant_values_come_back(ops):
    """All dims of every value alike (scale 0): the output is that number."""
    cache = ops.kv4_cache(2, 1)
    v = torch.full((1, 100, 1, 128), 0.375, dtype=torch.bfloat16, device="cuda")
    k = torch.randn(1, 100, 1, 128, device="cuda").to(torch.bfloat16)
    ops.kv4_append(k, v, cache, i32([[1, 0]]), i32([0]))
    q = torch.randn(1, 1, 8, 128, device="cuda").to(torch.bfloat16)
    got = ops.attention_kv4(q, cache, i32([[1, 0]]), i32([100]))
    assert ((got.float() - 0.375).abs() <= 0.375 * 2 ** -8).all()


def test_bad_pages_are_left_out(ops):
    rng = np.random.default_rng(14)
    cache = make_cache(rng, 4, 2)
    table = np.array([[0, 99, 1, -5], [2, 3, 2, 3]], np.int32)
    q = R.bf16_round(rng.standard_normal((2, 1, 4, 128)))
    got = ops.attention_kv4(bf(q), torch.from_numpy(cache).cuda(), i32(table), i32([256, 200]))
    assert status() == 8
    # the same sequence with the bad pages cut out
    ref, slack = R.attention(q, cache, np.array([[0, 1, 0, 0], [2, 3, 2, 3]]), [128, 200], None)
    err = np.abs(got.double().cpu().numpy() - ref)
    assert (err <= slack + 2 ** -8 * (np.abs(ref) + slack)).all()


def test_length_past_the_table_is_cut(ops):
    rng = np.random.default_rng(15)
    cache, table = make_cache(rng, 2, 1), np.array([[1, 0]], np.int32)
    q = bf(rng.standard_normal((1, 1, 8, 128)))
    a, b = (ops.attention_kv4(q, torch.from_numpy(cache).cuda(), i32(table), i32([n])) for n in (128, 10 ** 9))
    assert torch.equal(a, b)


@pytest.mark.parametrize("S", [1, 3, 80])
def test_a_bound_on_the_lengths(ops, S):
    """max_kv_len: any bound that holds gives the same rows (the forms may sum in
    another order); a length beyond it is cut."""
    rng = np.random.default_rng(18)
    table = np.arange(300, dtype=np.int32).reshape(2, 150)
    cache = torch.from_numpy(make_cache(rng, 300, 2)).cuda()
    q, n = bf(rng.standard_normal((2, S, 8, 128))), i32([130, 100])
    wide, close, cut = (ops.attention_kv4(q, cache, i32(table), k, max_kv_len=m) for m, k in ((None, n), (130, n), (100, n)))
    # two forms: weights and outputs rounded to bf16 at most, of values up to 8 times a scale of about 0.3
    assert (wide.float() - close.float()).abs().max() <= 8 * 2 ** -7
    assert torch.equal(cut, ops.attention_kv4(q, cache, i32(table[:, :2]), i32([100, 100]), max_kv_len=100))
    for bad in (0, 9601, -1):
        with pytest.raises(ValueError):
            ops.attention_kv4(q, cache, i32(table), n, max_kv_len=bad)


def test_far_pages(ops):
    """Byte offsets of the cache past 32 bits."""
    P = 530000  # 4.6 GB
    cache = torch.empty((P, 1, R.BLOB), dtype=torch.uint8, device="cuda")
    rng = np.random.default_rng(16)
    x = R.bf16_round(rng.standard_normal((1, 150, 1, 128)))
    far, near = i32([[P - 1, 500001, 3]]), i32([[0, 1, 2]])
    outs = []
    for t in (far, near):
        ops.kv4_append(bf(x), bf(x), cache, t, i32([0]))
        k, _ = ops.kv4_gather(cache, t, i32([0]), 150, i32([150]))
        outs.append((ops.attention_kv4(bf(x[:, :1]), cache, t, i32([150])), k))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


def test_views_streams_and_single_token_form(ops):
    rng = np.random.default_rng(17)
    lens = np.array([90, 300])
    table, P = make_table(rng, lens)
    cache = torch.from_numpy(make_cache(rng, P, 2)).cuda()
    q = bf(rng.standard_normal((2, 1, 8, 128)))
    want = ops.attention_kv4(q, cache, i32(table), i32(lens))
    row = torch.zeros(2, 1, 12, 128, dtype=torch.bfloat16, device="cuda")
    row[:, :, 2:10] = q
    assert torch.equal(ops.attention_kv4(row[:, :, 2:10], cache, i32(table), i32(lens)), want)
    assert torch.equal(ops.attention_kv4(q[:, 0], cache, i32(table), i32(lens)), want[:, 0])
    out = torch.zeros(2, 1, 12, 128, dtype=torch.bfloat16, device="cuda")
    ops.attention_kv4(q, cache, i32(table), i32(lens), out=out[:, :, 4:])
    assert torch.equal(out[:, :, 4:], want) and (out[:, :, :4] == 0).all()
    t, n = i32(table), i32(lens)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [ops.attention_kv4(q, cache, t, n) for _ in range(3)]
    s.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_refusals(ops):
    cache, t, n = ops.kv4_cache(4, 2), i32([[0, 1]]), i32([5])
    q = torch.zeros(1, 1, 4, 128, dtype=torch.bfloat16, device="cuda")
    for bad in (q.float(), q.half()):
        with pytest.raises(TypeError):
            ops.attention_kv4(bad, cache, t, n)
    for bad in (q[..., :64], q[:, :, :3], q.expand(2, 1, 4, 128), q.cpu(), torch.zeros(1, 1, 128, 4, dtype=torch.bfloat16, device="cuda").transpose(2, 3)):
        with pytest.raises(ValueError):
            ops.attention_kv4(bad, cache, t, n)
    with pytest.raises(TypeError):
        ops.attention_kv4(q, cache, t.long(), n)
    with pytest.raises(ValueError):
        ops.attention_kv4(q, cache, t, i32([5, 5]))
    with pytest.raises(ValueError):
        ops.attention_kv4(q, cache[:, :, :4096], t, n)
    k = torch.zeros(1, 3, 2, 128, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        ops.kv4_append(k, k[:, :2], cache, t, n)
    with pytest.raises(ValueError):
        ops.kv4_append(torch.zeros(1, 3, 2, 132, dtype=torch.bfloat16, device="cuda")[..., :128], k, cache, t, n)
    with pytest.raises(ValueError):
        ops.kv_pages_fork([cache, cache], t, n, i32([0, 0, 0, 0]), i32([0]))
    with pytest.raises(ValueError):
        ops.kv_pages_fork([cache], t, n, i32([0, 0, 0]), i32([0]))


# ---------------------------------------------------------------------------
# pages
# ---------------------------------------------------------------------------
def start_state(rng, B, M, P, pools, shapes):
    ref = R.Pages(np.full((B, M), -7, np.int32), np.zeros(B, np.int32), np.zeros(P, np.int32))
    data = [rng.integers(0, 256, (P,) + shapes[i % len(shapes)], dtype=np.uint8) for i in range(pools)]
    dev = dict(table=i32(ref.table), lens=i32(ref.lens), refs=i32(ref.refs), pools=[torch.from_numpy(d).cuda() for d in data])
    return ref, data, dev


def same_state(ref, data, dev):
    assert np.array_equal(dev["table"].cpu().numpy(), ref.table)
    assert np.array_equal(dev["lens"].cpu().numpy(), ref.lens)
    assert np.array_equal(dev["refs"].cpu().numpy(), ref.refs)
    for a, b in zip(dev["pools"], data):
        assert np.array_equal(a.cpu().numpy(), b)


@pytest.mark.parametrize("B, M, P, pools", [(1, 1, 1, 1), (5, 4, 13, 2), (33, 9, 200, 1), (130, 70, 5000, 2), (7, 40, 300, 66)])
def test_random_page_operations(ops, B, M, P, pools):
    rng = np.random.default_rng(B * 1000 + P)
    ref, data, dev = start_state(rng, B, M, P, pools, [(16,), (3, 48), (17, 1024)] if pools < 10 else [(32,)])
    seen = set()
    for step in range(14):
        what = ("extend", "extend", "fork", "compact")[step % 4] if step < 8 else rng.choice(["extend", "fork", "compact"])
        if what == "extend":
            new = rng.integers(0, max(2, 2 * P * 64 // B // 5), B) * (rng.random(B) < 0.7)
            new = np.minimum(new, np.maximum(0, M * 64 - ref.lens)) if rng.random() < 0.8 else new
            was = ref.lens.copy()
            want = ref.extend(new)
            start, st = ops.kv_pages_extend(dev["table"], dev["lens"], dev["refs"], i32(new))
            assert np.array_equal(start.cpu().numpy(), was)
        elif what == "fork":
            parent = np.arange(B)
            m = rng.random(B) < 0.5
            parent[m] = rng.integers(-1, B, int(m.sum()))
            want = ref.fork(parent, data)
            st = ops.kv_pages_fork(dev["pools"], dev["table"], dev["lens"], dev["refs"], i32(parent))
        else:
            want, remap = ref.compact(data)
            got, st = ops.kv_pages_compact(dev["pools"], dev["table"], dev["lens"], dev["refs"])
            assert np.array_equal(got.cpu().numpy(), remap)
        assert int(st) == want, what
        seen.add((what, want > 0))
        same_state(ref, data, dev)
    assert len({w for w, _ in seen}) == 3


def test_beams_that_change_places(ops):
    """Rows that are parents and children at once read the state before the call."""
    rng = np.random.default_rng(5)
    ref, data, dev = start_state(rng, 4, 5, 40, 2, [(64,)])
    ref.extend([100, 130, 64, 7])
    ops.kv_pages_extend(dev["table"], dev["lens"], dev["refs"], i32([100, 130, 64, 7]))
    for parent in ([1, 0, 3, 2], [3, 3, 3, 3], [0, 0, 1, 1], [-1, -1, 0, 3], [0, 0, -1, -1], [-1, -1, -1, -1]):
        want = ref.fork(parent, data)
        assert int(ops.kv_pages_fork(dev["pools"], dev["table"], dev["lens"], dev["refs"], i32(parent))) == want == 0
        same_state(ref, data, dev)
    assert (ref.refs == 0).all()


def test_page_calls_that_cannot_be_served_change_nothing(ops):
    rng = np.random.default_rng(6)
    ref, data, dev = start_state(rng, 3, 4, 5, 1, [(64,)])
    ref.extend([100, 100, 0])
    ops.kv_pages_extend(dev["table"], dev["lens"], dev["refs"], i32([100, 100, 0]))
    for new, want in (([0, 0, 129], 2), ([-1, 0, 0], -1), ([0, 0, 257], -1), ([2 ** 31 - 1, 0, 0], -1)):
        assert int(ops.kv_pages_extend(dev["table"], dev["lens"], dev["refs"], i32(new))[1]) == want == ref.extend(new)
        same_state(ref, data, dev)
    for parent, want in (([1, 0, 0], 2), ([3, 1, 2], -1), ([0, 1, -2], -1)):
        assert int(ops.kv_pages_fork(dev["pools"], dev["table"], dev["lens"], dev["refs"], i32(parent))) == want == ref.fork(parent, data)
        same_state(ref, data, dev)
    for name, at, bad in (("table", (1, 1), 5), ("table", (0, 0), -1), ("lens", (2,), -3), ("lens", (0,), 257)):
        good = dev[name][at].clone()
        dev[name][at], getattr(ref, name)[at] = bad, bad
        parent = [1, 0, 2] if name == "table" else [0, 0, 0] if bad < 0 else [1, 1, 2]
        assert int(ops.kv_pages_fork(dev["pools"], dev["table"], dev["lens"], dev["refs"], i32(parent))) == -1
        assert int(ops.kv_pages_compact(dev["pools"], dev["table"], dev["lens"], dev["refs"])[1]) == -1
        if name == "lens":
            assert int(ops.kv_pages_extend(dev["table"], dev["lens"], dev["refs"], i32([0, 0, 0]))[1]) == -1
        same_state(ref, data, dev)
        dev[name][at], getattr(ref, name)[at] = good, int(good)


@pytest.mark.parametrize("S", [1, 7, 64, 130])
def test_tokens_without_room_are_not_stored(ops, S):
    """Row 1 was long once; its table still names pages that are row 0's now."""
    H, old = 2, 192
    table, lens, refs = i32([[-1] * 8] * 2), i32([0, 0]), i32([0] * 6)
    cache = ops.kv4_cache(6, H)
    ops.kv_pages_extend(table, lens, refs, i32([0, old]))
    ops.kv_pages_fork([cache], table, lens, refs, i32([0, -1]))
    ops.kv_pages_extend(table, lens, refs, i32([6 * 64, 0]))
    assert table[0, :6].tolist() == [0, 1, 2, 3, 4, 5] and table[1, :3].tolist() == [0, 1, 2]
    k = torch.randn(2, S, H, 128, device="cuda").to(torch.bfloat16)
    start, lack = ops.kv_pages_extend(table, lens, refs, i32([0, S]))
    assert int(lack) == -(-S // 64) and start.tolist() == [384, 0] and lens.tolist() == [384, 0]
    ops.kv4_append(k, k, cache, table, start, new_len=i32([0, S]), kv_len=lens)
    assert not cache.any() and status() == 0
    # and up to the length, not past it
    ops.kv4_append(k, k, cache, table, i32([0, 0]), new_len=i32([S, 0]), kv_len=i32([S // 2, 0]))
    want = ops.kv4_cache(6, H)
    ops.kv4_append(k, k, want, table, i32([0, 0]), new_len=i32([S // 2, 0]))
    assert torch.equal(cache, want) and status() == 0


def test_lengths_that_double(ops):
    """The lengths themselves as the number of new tokens."""
    table, lens, refs = i32([[-1] * 40] * 40), i32([5 * i for i in range(40)]), i32([0] * 400)
    for b in range(40):
        for c in range(-(-5 * b // 64)):
            p = int((refs > 0).sum())
            table[b, c], refs[p] = p, 1
    start, lack = ops.kv_pages_extend(table, lens, refs, lens)
    assert int(lack) == 0 and start.tolist() == [5 * i for i in range(40)] and lens.tolist() == [10 * i for i in range(40)]
    assert int((refs == 1).sum()) == sum(-(-10 * i // 64) for i in range(40))


def test_a_tensor_is_no_list_of_pools(ops):
    pool = torch.zeros(4, 4, 8704, dtype=torch.uint8, device="cuda")
    with pytest.raises(TypeError):
        ops.kv_pages_fork(pool, i32([[0] * 4]), i32([0]), i32([0] * 4), i32([0]))
    with pytest.raises(TypeError):
        ops.kv_pages_compact(pool, i32([[0] * 4]), i32([0]), i32([0] * 4))


def test_empty_batches_and_pools(ops):
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    t = torch.empty(0, 3, dtype=torch.int32, device="cuda")
    start, st = ops.kv_pages_extend(t, e, i32([0, 0]), e)
    assert start.numel() == 0 and int(st) == 0
    assert int(ops.kv_pages_fork([], t, e, i32([0, 1]), e)) == 0
    pool = torch.arange(32, dtype=torch.uint8, device="cuda").view(2, 16)
    remap, live = ops.kv_pages_compact([pool], t, e, i32([0, 1]))  # a page held outside the table
    assert remap.tolist() == [-1, 0] and int(live) == 1 and pool[0].tolist() == list(range(16, 32))
    cache = ops.kv4_cache(1, 1)
    assert ops.attention_kv4(torch.empty(0, 1, 4, 128, dtype=torch.bfloat16, device="cuda"), cache, t, e).shape == (0, 1, 4, 128)
    assert ops.attention_kv4(torch.empty(2, 0, 4, 128, dtype=torch.bfloat16, device="cuda"), cache, i32([[0], [0]]), i32([1, 1])).shape == (2, 0, 4, 128)
    assert ops.attention_kv4(torch.ones(2, 1, 4, 128, dtype=torch.bfloat16, device="cuda"), cache, i32([[0], [0]]), i32([0, 0])).abs().sum() == 0


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
def test_a_serving_run(ops):
    """Two requests; one branches into three beams that go on with tokens of
    their own; requests end, pages are compacted; every step's attention is
    that over the tokens the sequence has had, and compaction changes no bit."""
    rng = np.random.default_rng(21)
    B, M, P, H, Hq, layers = 5, 6, 24, 2, 8, 2
    pools = [ops.kv4_cache(P, H) for _ in range(layers)]
    table, lens, refs = i32(np.full((B, M), -1)), i32(np.zeros(B)), i32(np.zeros(P))
    past = [[np.zeros((0, H, 128)), np.zeros((0, H, 128))] for _ in range(B)]

    def step(new):
        S = max(new)
        k, v = (R.bf16_round(rng.standard_normal((B, S, H, 128))) for _ in range(2))
        start, st = ops.kv_pages_extend(table, lens, refs, i32(new))
        for pool in pools:
            ops.kv4_append(bf(k), bf(v), pool, table, start, i32(new))
        for b in range(B):
            past[b] = [np.concatenate([past[b][0], k[b, : new[b]]]), np.concatenate([past[b][1], v[b, : new[b]]])]
        assert int(st) == 0

    def attend(pool):
        q = R.bf16_round(rng.standard_normal((B, 1, Hq, 128)))
        got = ops.attention_kv4(bf(q), pool, table, lens, start_pos=lens - 1)
        for b in range(B):
            blob = np.zeros((R.pages_of(len(past[b][0])) or 1, H, R.BLOB), np.uint8)
            for i, (k, v) in enumerate(zip(*past[b])):
                for h in range(H):
                    R.put_token(blob[i // 64, h], i % 64, k[h], v[h])
            ref, slack = R.attention(q[b: b + 1], blob, np.arange(len(blob))[None], [len(past[b][0])], None)
            assert (np.abs(got[b: b + 1].double().cpu().numpy() - ref) <= slack + 2 ** -8 * (np.abs(ref) + slack)).all()
        return bf(q), got

    def fork(parent):
        assert int(ops.kv_pages_fork(pools, table, lens, refs, i32(parent))) == 0
        past[:] = [[x.copy() for x in past[p]] if p >= 0 else [np.zeros((0, H, 128))] * 2 for p in parent]

    step([130, 70, 0, 0, 0])
    fork([0, 1, 0, 0, -1])
    for _ in range(3):
        step([1, 1, 1, 1, 0])
    attend(pools[1])
    fork([2, 1, 2, 0, 1])   # beams reordered, the second request branches too
    step([1, 60, 1, 1, 2])
    attend(pools[0])
    fork([-1, 1, 2, -1, 4])
    q, before = attend(pools[0])
    remap, live = ops.kv_pages_compact(pools, table, lens, refs)
    n = int(live)
    assert (refs[:n] > 0).all() and (refs[n:] == 0).all()
    assert torch.equal(ops.attention_kv4(q, pools[0], table, lens, start_pos=lens - 1), before)
    attend(pools[1])
    assert status() == 0


def test_a_captured_decode_step(ops):
    """Growing, storing and attending in one CUDA graph, replayed over a page
    border, next to a second captured graph and eager calls."""
    rng = np.random.default_rng(22)
    B, M, P, H, Hq = 3, 3, 9, 2, 8
    graphs = []
    for _ in range(2):
        st = dict(pool=ops.kv4_cache(P, H), table=i32(np.full((B, M), -1)), lens=i32(np.zeros(B)), refs=i32(np.zeros(P)),
                  one=i32([1, 1, 0]), k=torch.zeros(B, 1, H, 128, dtype=torch.bfloat16, device="cuda"),
                  q=torch.zeros(B, 1, Hq, 128, dtype=torch.bfloat16, device="cuda"))

        def step(st=st):
            start, status = ops.kv_pages_extend(st["table"], st["lens"], st["refs"], st["one"])
            ops.kv4_append(st["k"], st["k"], st["pool"], st["table"], start, st["one"])
            return ops.attention_kv4(st["q"], st["pool"], st["table"], st["lens"], start_pos=start), status

        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        for n in ("lens", "refs"):
            st[n].zero_()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            st["out"], st["status"] = step()
        graphs.append((g, st))
    past = [[] for _ in graphs]
    for i in range(66):
        for j, (g, st) in enumerate(graphs):
            k, q = R.bf16_round(rng.standard_normal((B, 1, H, 128))), R.bf16_round(rng.standard_normal((B, 1, Hq, 128)))
            st["k"].copy_(bf(k))
            st["q"].copy_(bf(q))
            g.replay()
            past[j].append(k)
            if i in (0, 62, 63, 64, 65):
                assert st["lens"].tolist() == [i + 1, i + 1, 0] and int(st["status"]) == 0
                cache = st["pool"].cpu().numpy()
                ref, slack = R.attention(q, cache, st["table"].cpu().numpy(), [i + 1, i + 1, 0], None)
                err = np.abs(st["out"].double().cpu().numpy() - ref)
                assert (err <= slack + 2 ** -8 * (np.abs(ref) + slack)).all()
    for (g, st), hist in zip(graphs, past):
        k, _ = ops.kv4_gather(st["pool"], st["table"], i32(np.zeros(B)), 66, st["lens"])
        u, s, m = R.quantise(np.concatenate(hist, 1))
        assert np.array_equal(k[:2].cpu().numpy(), (m[..., None] + s[..., None] * u).astype(np.float32)[:2])


def test_attention_agrees_with_the_bf16_cache(ops):
    """Next to the framework's own decode attention: with keys and values that
    4 bits hold exactly, both give the same to bf16's rounding."""
    from metalbench_b200 import _lib
    rng = np.random.default_rng(23)
    B, Hq, Hkv, L = 3, 8, 2, 200
    lo = rng.integers(-6, 0, (B, L, Hkv, 1)).astype(np.float64)
    u = rng.integers(0, 16, (B, L, Hkv, 128)).astype(np.float64)
    u[..., 0], u[..., 1] = 0, 15
    kv = [(lo + u) * 2.0 ** -3, (lo + u[..., ::-1]) * 2.0 ** -2]
    M = R.pages_of(L)
    table = np.arange(B * M, dtype=np.int32).reshape(B, M)
    bfc = [np.zeros((B * M, Hkv, 64, 128)) for _ in kv]
    for c, x in zip(bfc, kv):
        for b in range(B):
            for p in range(L):
                c[table[b, p // 64], :, p % 64] = x[b, p]
    cache = ops.kv4_cache(B * M, Hkv)
    ops.kv4_append(bf(kv[0]), bf(kv[1]), cache, i32(table), i32([0] * B))
    q = bf(R.bf16_round(rng.standard_normal((B, 1, Hq, 128))))
    lens = np.array([200, 64, 1])
    got = ops.attention_kv4(q, cache, i32(table), i32(lens))
    kc, vc = (bf(c) for c in bfc)
    out = torch.empty(B, Hq * 128, dtype=torch.bfloat16, device="cuda")
    t, n = i32(table), i32(lens)
    nb = _lib.lib().mb_attention_decode_workspace_bytes(B, Hq, Hkv, L)
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
    _lib.call("mb_attention_decode_bf16", q.data_ptr(), Hq * 128, kc.data_ptr(), vc.data_ptr(), t.data_ptr(), M, n.data_ptr(),
              L, B, Hq, Hkv, 128, out.data_ptr(), Hq * 128, ws.data_ptr(), nb, torch.cuda.current_stream().cuda_stream)
    # each side: its weights rounded (bf16 2^-8, fp16 2^-11) and its output (2^-8); values up to 2.25
    bound = (2 ** -8 + 2 ** -10) * 2.25 + 2 * 2 ** -8 * 2.25
    assert (got.view(B, -1).float() - out.float()).abs().max() <= bound
