"""The 8-bit append at the limits of its arguments: positions at the ends of the 32-bit range, sizes that no index may pass."""
import numpy as np
import pytest

import view_reference as R
from test_q8_cache import _append_args, _append_reference, _check_append, _refusal, _rotate32, _rope_tables, _run_append


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [0, 1])
@pytest.mark.parametrize("block_size,d", [(16, 128), (16, 64), (1, 40), (5, 8)])
def test_append_with_positions_at_the_ends_of_the_range(compute, cache_dtype, block_size, d):
    """Positions that no table can hold are skipped and reported, the sequences beside them are written as ever."""
    from granite_b200.capi import ErrorCode
    rng = np.random.default_rng(block_size)
    positions = np.array([2 ** 31 - 1, 3, 2 ** 31 - 200, -(2 ** 31), 0, 2 ** 30, -1], np.int32)
    hkv, n, limit = 2, 300, 320
    pages = -(-limit // block_size)
    tables = np.arange(len(positions) * pages, dtype=np.int32).reshape(len(positions), pages)
    blocks = tables.size
    pools = [R.random_pool(rng, blocks, block_size, hkv, d, cache_dtype) for _ in range(2)]
    codes, scales = [p[0] for p in pools], [p[1] for p in pools]
    k, v = (rng.standard_normal((len(positions), n, hkv, d), dtype=np.float32) for _ in range(2))
    q = rng.standard_normal((len(positions), n, 2, d), dtype=np.float32)
    cos, sin = _rope_tables(limit, d)
    got = _run_append(compute, q, k, v, cos, sin, codes, scales, tables, positions, block_size, cache_dtype)
    assert got[3] is not None and got[3].code == ErrorCode.InvalidArgument
    where = positions[:, None].astype(np.int64) + np.arange(n)
    ok, at = ((where >= 0) & (where < limit))[:, :, None, None], np.clip(where, 0, limit - 1)
    want_codes, want_scales = [c.copy() for c in codes], [s.copy() for s in scales]
    for x, c, s in ((_rotate32(k, cos[at][:, :, None], sin[at][:, :, None]), want_codes[0], want_scales[0]), (v, want_codes[1], want_scales[1])):
        _append_reference(x, c, s, tables, positions, block_size, cache_dtype, limit)
    _check_append(got, (want_codes, want_scales))
    assert np.array_equal(got[0], np.where(ok, _rotate32(q, cos[at][:, :, None], sin[at][:, :, None]), q))
    compute.sync()


@pytest.mark.parametrize("block_size,head_dim", [(1 << 25, 256), ((1 << 31) - 1, 8), (1 << 26, 128), ((1 << 30) - 32768, 8)])
def test_a_page_whose_pieces_pass_32_bits_is_refused(block_size, head_dim):
    """Rows of a page times its four-element pieces are counted in 32 bits; the last case is the first size that is refused."""
    from granite_b200 import capi
    args = _append_args(block_size=block_size, head_dim=head_dim, max_blocks_per_seq=1, num_blocks=1)
    got, text = _refusal(capi.lib.granite_cuda_rope_paged_kv_cache_append_q8, *args)
    assert got.name == "InvalidArgument" and "block_size" in text
    got, text = _refusal(capi.lib.granite_cuda_rope_paged_kv_cache_append_q8, *_append_args(block_size=(1 << 30) - 32769, head_dim=8))
    assert got.name == "NullPointer" and "compute object" in text  # nothing left to refuse but the missing object


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [0, 1])
@pytest.mark.parametrize("block_size,d", [(16, 128), (16, 64), (8, 40)])
@pytest.mark.parametrize("magnitude", [2.0 ** -117, 2.0 ** -110, 2.0 ** -100, 2.0 ** -80, 2.0 ** 100, 2.0 ** 126])
def test_append_of_tiny_and_huge_values_writes_the_defined_bytes(compute, cache_dtype, block_size, d, magnitude):
    """round(x / scale) to the last bit at both ends of the range, halves of a step among the values (where the quotient's last bit decides):
    scales down to the smallest normal number, and up to a 127th of the largest."""
    rng = np.random.default_rng(d)
    hkv, n, batch = 4, 40, 3
    qmax = R.QMAX[cache_dtype]
    positions = np.array([0, 5, 17], np.int32)
    pages = -(-(n + 17) // block_size)
    tables = np.arange(batch * pages, dtype=np.int32).reshape(batch, pages)
    pools = [R.random_pool(rng, tables.size, block_size, hkv, d, cache_dtype) for _ in range(2)]
    codes, scales = [p[0] for p in pools], [(p[1] * magnitude / qmax).astype(np.float32) for p in pools]
    # every value a whole or half number of steps of a page's likely scale, give or take a unit in the last place
    top = (rng.uniform(1, 1.9, (batch, n, hkv, 1)) * magnitude).astype(np.float32)
    x = ((rng.integers(-2 * int(qmax), 2 * int(qmax) + 1, (batch, n, hkv, d)) / (2 * qmax)).astype(np.float32) * top).astype(np.float32)
    x[..., 0] = top[..., 0]
    x = np.nextafter(x, np.float32(0) + rng.integers(-1, 2, x.shape).astype(np.float32) * np.float32(3e38))
    v = x[:, ::-1].copy()
    cos, sin = np.ones((n + 20, d // 2), np.float32), np.zeros((n + 20, d // 2), np.float32)
    got = _run_append(compute, None, x, v, cos, sin, codes, scales, tables, positions, block_size, cache_dtype)
    assert got[3] is None
    want_codes, want_scales = [c.copy() for c in codes], [s.copy() for s in scales]
    _append_reference(_rotate32(x, np.float32(1), np.float32(0)), want_codes[0], want_scales[0], tables, positions, block_size, cache_dtype, n + 20)
    _append_reference(v, want_codes[1], want_scales[1], tables, positions, block_size, cache_dtype, n + 20)
    _check_append(got, (want_codes, want_scales))
