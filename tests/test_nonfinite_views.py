"""What is not finite and is seen comes out as not finite, in its own row and head and nowhere else: for the 8-bit and windowed calls on the
shapes of the tuned kernels and on those of the plain one alike."""
import numpy as np
import pytest

import view_reference as R
from test_q8_cache import _dev, _table

DEV = "cuda:0"
SHAPES = [(8, 2, 128, 16), (4, 2, 64, 16), (4, 2, 40, 16), (4, 2, 128, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d,block_size", SHAPES)
@pytest.mark.parametrize("cache_dtype", [None, 0, 1])
@pytest.mark.parametrize("prefill", [False, True])
def test_a_query_that_is_not_finite_gives_no_finite_output(compute, hq, hkv, d, block_size, cache_dtype, prefill):
    import torch
    rng = np.random.default_rng(d)
    n, rows, window, sinks = 150, 20, 60, 3
    tables, blocks = _table(rng, [n], block_size)
    tables = np.repeat(tables, rows, 0)  # decode: the same pages for every sequence, which are of growing length
    lens = np.arange(n - rows + 1, n + 1, dtype=np.int32)
    if cache_dtype is None:
        k, v = (rng.standard_normal((blocks * block_size, hkv, d)).astype(np.float16) for _ in range(2))
        kv, vv = k.astype(np.float64), v.astype(np.float64)
        scales = ()
    else:
        (k, ks), (v, vs) = (R.random_pool(rng, blocks, block_size, hkv, d, cache_dtype) for _ in range(2))
        kv, vv = R.pool_values(k, ks, cache_dtype, block_size), R.pool_values(v, vs, cache_dtype, block_size)
        scales = (_dev(ks), _dev(vs))
    q = rng.standard_normal((rows, hq, d), dtype=np.float32)
    bad = q.copy()
    bad[2, 1], bad[7, 3, 5], bad[11, 0, 0] = np.nan, np.nan, np.inf
    spoilt = ~np.isfinite(bad).all(-1)
    want, bound = R.attend(q.astype(np.float64), R.rows_of(kv, tables[0], n, block_size), R.rows_of(vv, tables[0], n, block_size), lens - 1, d ** -0.5, window, sinks)
    out = torch.zeros(q.shape, device=DEV)
    args = [_dev(bad), _dev(k), _dev(v), *scales]
    extra = {} if cache_dtype is None else dict(cache_dtype=cache_dtype)
    if prefill:
        fn = compute.paged_prefill_attention_window if cache_dtype is None else compute.paged_prefill_attention_q8
        fn(*args, _dev(tables[:1]), out, hq, hkv, rows, n - rows, d, block_size, tables.shape[1], blocks, d ** -0.5, window=window, sinks=sinks, **extra)
    else:
        fn = compute.batched_paged_attention_decode_window if cache_dtype is None else compute.batched_paged_attention_decode_q8
        fn(*args, _dev(tables), _dev(lens), out, rows, hq, hkv, d, block_size, tables.shape[1], d ** -0.5, num_blocks=blocks, window=window, sinks=sinks, **extra)
    compute.sync()
    got = out.cpu().numpy()
    assert not np.isfinite(got[spoilt]).any()
    got[spoilt] = want[spoilt]
    R.assert_close(got, want, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d,block_size", SHAPES)
@pytest.mark.parametrize("which", ["k", "v", "k scale", "v scale"])
def test_a_visible_key_that_is_not_finite_is_not_passed_over(compute, hq, hkv, d, block_size, which):
    """A NaN in a visible key (an e4m3 code) or in the scale of its page: the rows of its KV head are NaN, the other heads' come out right."""
    import torch
    rng = np.random.default_rng(d + 1)
    n = 150
    tables, blocks = _table(rng, [n], block_size)
    (k, ks), (v, vs) = (tuple(x.copy() for x in R.random_pool(rng, blocks, block_size, hkv, d, 1)) for _ in range(2))
    kv, vv = R.pool_values(k, ks, 1, block_size), R.pool_values(v, vs, 1, block_size)
    q = rng.standard_normal((1, hq, d), dtype=np.float32)
    want, bound = R.attend(q.astype(np.float64), R.rows_of(kv, tables[0], n, block_size), R.rows_of(vv, tables[0], n, block_size), [n - 1], d ** -0.5)
    page = tables[0, 70 // block_size]
    if which == "k":
        k[page * block_size + 70 % block_size, 1, 3] = 0x7F
    elif which == "v":
        v[page * block_size + 70 % block_size, 1] = 0x7F
    else:
        (ks if which == "k scale" else vs)[page, 1] = np.nan
    out = torch.zeros(q.shape, device=DEV)
    compute.batched_paged_attention_decode_q8(_dev(q), _dev(k), _dev(v), _dev(ks), _dev(vs), _dev(tables), _dev(np.array([n], np.int32)), out, 1, hq, hkv, d,
                                              block_size, tables.shape[1], d ** -0.5, num_blocks=blocks, cache_dtype=1)
    compute.sync()
    got = out.cpu().numpy()
    g = hq // hkv
    assert np.isnan(got[:, g:2 * g]).all()
    R.assert_close(got[:, :g], want[:, :g], bound[:, :g])
