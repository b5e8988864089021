"""The decoder layer and the stack over a 4-bit cache (PagedKV4Cache), against
the oracle run on the values that the cache holds. Gate as in test_decoder_gpu:
>= 99 % of elements within 2e-2*|b| + 2e-2*rms(b), max |a-b| <= 0.1*rms(b); what
the new tokens' own rounding to 4 bits adds is derived where it matters."""
import numpy as np
import pytest

import _kv4ref as R
import oracle.ops as O
from test_decoder_gpu import _bf, _check, _layer, _np, _weights

pytestmark = pytest.mark.gpu

D, H, Hkv, FF, BASE = 512, 4, 2, 512, 10000.0


def _i32(x):
    import torch
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).cuda()


def _held(cache, i, L):
    """What layer i's cache holds: k, v [B, Hkv, L, 128] float32."""
    from metalbench_b200 import ops
    B = cache.batch
    k, v = ops.kv4_gather(cache.pools[i], cache.block_table, _i32([0] * B), L, cache.seq_len)
    return (x.permute(0, 2, 1, 3).cpu().numpy() for x in (k, v))


@pytest.mark.parametrize("B, S", [(2, 70), (3, 1), (1, 200)])
def test_layer_stores_the_quantised_keys_and_values(B, S):
    """The same layer over the bf16 cache writes the same bf16 keys and values;
    the 4-bit one holds exactly their quantised values."""
    import torch
    from metalbench_b200.decoder import PagedKV4Cache, PagedKVCache
    rng = np.random.default_rng(S)
    layer = _layer(torch, _weights(rng, D, H, Hkv, FF), D, H, Hkv, FF, BASE)
    x = _bf(torch, rng.standard_normal((B, S, D)))
    wide = PagedKVCache(B, S, Hkv)
    layer(x, wide, _i32([0] * B))
    cache = PagedKV4Cache(B, 256, Hkv)
    start = cache.extend(_i32([S] * B))
    layer(x, cache.layer(0), start)
    assert int(cache.status) == 0 and cache.seq_len.tolist() == [S] * B
    for got, pages in zip(_held(cache, 0, S), (wide.k, wide.v)):
        rows = _np(torch, pages).reshape(B, -1, Hkv, 64, 128).transpose(0, 2, 1, 3, 4).reshape(B, Hkv, -1, 128)[:, :, :S]
        u, s, m = R.quantise(rows)
        assert np.array_equal(got, (m[..., None] + s[..., None] * u).astype(np.float32))


def test_decode_over_a_held_cache_matches_oracle():
    """One token a sequence over 200, 64 and 130 held ones: the oracle gets the
    values that the 4 bits stand for. The new token's own rounding moves an
    output by its weight, about 1/64 at most, times half a code step."""
    import torch
    from metalbench_b200.decoder import PagedKV4Cache
    rng = np.random.default_rng(11)
    W = _weights(rng, D, H, Hkv, FF)
    layer = _layer(torch, W, D, H, Hkv, FF, BASE)
    lens = [200, 64, 130]
    cache = PagedKV4Cache(3, 256, Hkv, num_pages=14)
    start = cache.extend(_i32(lens))
    k, v = (_bf(torch, rng.standard_normal((3, 200, Hkv, 128)) * 0.5) for _ in range(2))
    cache.append(0, k, v, start, _i32(lens))
    past = [list(_held(cache, 0, 200))]
    x = O.round_bf16(rng.standard_normal((3, 1, D)).astype(np.float32))
    start = cache.extend(_i32([1, 1, 1]))
    got = _np(torch, layer(_bf(torch, x), cache.layer(0), start))
    for b, L in enumerate(lens):
        ref = O.decoder_layer(x[b: b + 1], *W, H=H, H_kv=Hkv, base=BASE, causal=True,
                              k_past=past[0][0][b: b + 1, :, :L], v_past=past[0][1][b: b + 1, :, :L])
        _check(got[b: b + 1], ref)


def test_padded_step_equals_single_tokens():
    """Three tokens of one sequence and one of another in a padded call, and one
    by one: the same cache and the same rows."""
    import torch
    from metalbench_b200.decoder import PagedKV4Cache
    rng = np.random.default_rng(12)
    layer = _layer(torch, _weights(rng, D, H, Hkv, FF), D, H, Hkv, FF, BASE)
    x = _bf(torch, rng.standard_normal((2, 3, D)))
    k, v = (_bf(torch, rng.standard_normal((2, 63, Hkv, 128))) for _ in range(2))
    outs = []
    for padded in (True, False):
        cache = PagedKV4Cache(2, 192, Hkv)
        cache.append(0, k, v, cache.extend(_i32([63, 63])))
        if padded:
            new = _i32([3, 1])
            y = layer(x, cache.layer(0), cache.extend(new), new_len=new)
            rows = [y[0], y[1, :1]]
        else:
            ys = []
            for s, new in enumerate(([1, 1], [1, 0], [1, 0])):
                ys.append(layer(x[:, s: s + 1].contiguous(), cache.layer(0), cache.extend(_i32(new)), new_len=_i32(new)))
            rows = [torch.cat([y[0] for y in ys]), ys[0][1]]
        assert cache.seq_len.tolist() == [66, 64] and int(cache.status) == 0
        outs.append((rows, list(_held(cache, 0, 66))))
    for a, b in zip(outs[0][0], outs[1][0]):
        _check(_np(torch, a), _np(torch, b))
    # the tokens that were there before are the same bits; new ones went through differently tiled
    # GEMMs, whose bf16 outputs may differ in their last place and move a code by one
    for a, b in zip(outs[0][1], outs[1][1]):
        assert np.array_equal(a[:, :, :63], b[:, :, :63])
        assert np.abs(a - b).max() <= 1.01 * (np.abs(b).max() * 2 / 15)


def test_stack_over_four_bits_in_a_graph():
    """Two layers, a captured decode step over 100 held tokens, replayed; then a
    beam fork and a compaction between steps."""
    import torch
    from metalbench_b200.decoder import DecoderConfig
    from metalbench_b200.stack import DecoderStack
    rng = np.random.default_rng(13)
    B, L, n = 3, 100, 2
    Ws = [_weights(rng, D, H, Hkv, FF) for _ in range(n)]
    st = DecoderStack(DecoderConfig(D, H, Hkv, FF, rope_base=BASE), n, B, 256,
                      weights=[[_bf(torch, w) for w in W] for W in Ws], kv_bits=4)
    st.fill_cache_random(L)
    cache = st.kv4
    assert cache.seq_len.tolist() == [L] * B and int(cache.status) == 0

    def want(x, length):
        for i, W in enumerate(Ws):
            k, v = _held(cache, i, length)
            x = O.decoder_layer(x, *W, H=H, H_kv=Hkv, base=BASE, causal=True, k_past=k, v_past=v)
        return x

    x = O.round_bf16(rng.standard_normal((B, 1, D)).astype(np.float32))
    ref = want(x, L)
    start = cache.extend(_i32([1] * B))
    st.capture_decode(_bf(torch, x), start, L + 1)
    _check(_np(torch, st.replay()), ref)
    cache.fork(_i32([1, 1, 0]))
    assert int(cache.status) == 0
    remap, live = cache.compact()
    assert int(live) == int((cache.page_refs > 0).sum()) and (cache.page_refs[int(live):] == 0).all()
    x2 = O.round_bf16(rng.standard_normal((B, 1, D)).astype(np.float32))
    ref = want(x2, L + 1)
    start = cache.extend(_i32([1] * B))
    _check(_np(torch, st.forward(_bf(torch, x2), start)), ref)
    st.close()


def test_refusals():
    import torch
    from metalbench_b200.decoder import PagedKV4Cache, PagedKVCache
    rng = np.random.default_rng(14)
    layer = _layer(torch, _weights(rng, D, H, Hkv, FF), D, H, Hkv, FF, BASE)
    x = _bf(torch, rng.standard_normal((2, 1, D)))
    with pytest.raises(ValueError):
        layer(x, PagedKV4Cache(3, 64, Hkv).layer(0), _i32([0, 0]))
    with pytest.raises(ValueError):
        layer(x, PagedKV4Cache(2, 64, Hkv + 1).layer(0), _i32([0, 0]))
    with pytest.raises(ValueError):
        layer(x, PagedKV4Cache(2, 64, Hkv).layer(0), _i32([0, 0]), new_len=_i32([1]))
    with pytest.raises(ValueError):
        layer(x, PagedKVCache(2, 64, Hkv), _i32([0, 0]), new_len=_i32([1, 1]))
    with pytest.raises(ValueError):
        PagedKV4Cache(0, 64, Hkv)
    cache = PagedKV4Cache(2, 128, Hkv, num_pages=1)
    cache.extend(_i32([1, 1]))
    assert int(cache.status) == 1 and cache.seq_len.tolist() == [0, 0]
