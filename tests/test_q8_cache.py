"""The 8-bit paged cache: appending with the rotation, decode and chunked prefill over it, against plain 64-bit forms."""
import ctypes as C

import numpy as np
import pytest

import view_reference as R

DEV = "cuda:0"


def _table(rng, lens, block_size, spare=2):
    """Block tables that deal a permutation of the pool to the sequences; -1 behind the last page."""
    pages = (np.asarray(lens, np.int64) + block_size - 1) // block_size
    num = int(pages.sum()) + spare
    perm = rng.permutation(num).astype(np.int32)
    tables = np.full((len(pages), max(int(pages.max(initial=1)), 1)), -1, np.int32)
    off = 0
    for b, n in enumerate(pages):
        tables[b, :n] = perm[off:off + n]
        off += int(n)
    return tables, num


def _dev(x, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x))
    return t.to(DEV) if dtype is None else t.to(DEV, dtype)


def _rope_tables(n, d):
    a = np.arange(n)[:, None] * 10000.0 ** (-np.arange(0, d, 2) / d)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def _rotate32(x, cos, sin):
    """The rotation in the framework's fp32 arithmetic: products and sums rounded separately."""
    a, b = x[..., 0::2], x[..., 1::2]
    out = np.empty_like(x)
    out[..., 0::2] = a * cos - b * sin
    out[..., 1::2] = a * sin + b * cos
    return out


def _append_reference(x, codes, scales, tables, positions, block_size, cache_dtype, limit):
    """The append's definition on one of K and V ([B, n, Hkv, D], rotated), in fp32 where a value is stored or divided: the
    results are then the exact bytes.  Returns what would have been reported as non-finite."""
    qmax = np.float32(R.QMAX[cache_dtype])
    dropped = not np.isfinite(x).all()
    x = np.where(np.isfinite(x), x, np.float32(0))
    for b in range(x.shape[0]):
        lo, hi = max(int(positions[b]), 0), min(int(positions[b]) + x.shape[1], limit)
        at = lo
        while at < hi:
            end = min((at // block_size + 1) * block_size, hi)
            page, r0 = int(tables[b, at // block_size]), at % block_size
            if page >= 0:
                rows = x[b, at - int(positions[b]):end - int(positions[b])]
                mine = codes[page * block_size:(page + 1) * block_size]
                for h in range(x.shape[2]):
                    need = np.float32(np.abs(rows[:, h]).max()) / qmax
                    need = need if need >= np.float32(2.0 ** -126) else np.float32(0)
                    before = scales[page, h] if r0 else np.float32(0)
                    after = max(before, need)
                    if after > before and r0:
                        old = R.decode_codes(mine[:r0, h], cache_dtype).astype(np.float32) * (before / after)
                        mine[:r0, h] = R.encode(old.astype(np.float64), cache_dtype)
                    new = rows[:, h] / after if after > 0 else np.zeros_like(rows[:, h])
                    mine[r0:r0 + end - at, h] = R.encode(new.astype(np.float64), cache_dtype) if after > 0 else 0
                    scales[page, h] = after
            at = end
    return dropped


def _run_append(compute, q, k, v, cos, sin, codes, scales, tables, positions, block_size, cache_dtype, start_pos=0):
    """Device copies of everything, one call; the updated arrays."""
    b, n, hkv, d = k.shape
    qd = _dev(q) if q is not None else None
    kd, vd, kc, vc, ks, vs = (_dev(t) for t in (k, v, codes[0], codes[1], scales[0], scales[1]))
    cd, sd, td = _dev(cos), _dev(sin), _dev(tables)
    pd = _dev(positions) if positions is not None else None
    compute.rope_paged_kv_cache_append_q8(qd, kd, vd, cd, sd, kc, vc, ks, vs, td, pd, b, n, q.shape[2] if q is not None else 0, hkv, d,
                                          block_size, tables.shape[1], scales[0].shape[0], cos.shape[0], cache_dtype, start_pos)
    err = None
    try:
        compute.sync()
    except Exception as e:  # the status is the test's business
        err = e
    assert np.array_equal(kd.cpu().numpy(), k, equal_nan=True) and np.array_equal(vd.cpu().numpy(), v, equal_nan=True)  # inputs untouched
    return (qd.cpu().numpy() if q is not None else None, [kc.cpu().numpy(), vc.cpu().numpy()], [ks.cpu().numpy(), vs.cpu().numpy()], err)


def _check_append(got, want):
    q, codes, scales, err = got
    assert np.array_equal(scales[0].view(np.uint32), want[1][0].view(np.uint32))
    assert np.array_equal(scales[1].view(np.uint32), want[1][1].view(np.uint32))
    for g, w in zip(codes, want[0]):
        # a negative value that rounds to zero has e4m3 code 0x80 on both sides
        assert np.array_equal(g, w), f"{(g != w).sum()} codes differ"


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [0, 1])
@pytest.mark.parametrize("batch,new_len,hq,hkv,d,block_size,max_pos", [
    (64, 1, 32, 8, 128, 16, 400), (5, 5, 32, 4, 128, 16, 60), (3, 37, 16, 2, 64, 16, 40), (1, 300, 8, 8, 128, 16, 0),
    (2, 16, 0, 1, 128, 16, 16), (7, 3, 4, 2, 40, 16, 50), (3, 21, 6, 3, 256, 32, 70), (4, 9, 8, 8, 8, 5, 30), (2, 33, 5, 1, 128, 64, 64)])
def test_append_writes_the_defined_bytes(compute, cache_dtype, batch, new_len, hq, hkv, d, block_size, max_pos):
    rng = np.random.default_rng(batch * 1000 + new_len + d)
    positions = rng.integers(0, max_pos + 1, batch).astype(np.int32)
    positions[0] = min(max_pos, block_size - 1)  # the page's last row, where there is room for one
    tables, blocks = _table(rng, positions + new_len, block_size)
    pools = [R.random_pool(rng, blocks, block_size, hkv, d, cache_dtype) for _ in range(2)]
    codes, scales = [p[0] for p in pools], [p[1] for p in pools]
    q = rng.standard_normal((batch, new_len, hq, d), dtype=np.float32) if hq else None
    # token magnitudes over a factor of 100, so that scales grow in some pages and stay in others; a head of zeros
    k, v = (rng.standard_normal((batch, new_len, hkv, d), dtype=np.float32) *
            (10.0 ** rng.uniform(-1, 1, (batch, new_len, 1, 1))).astype(np.float32) for _ in range(2))
    v[-1, :, 0] = 0
    k[0, 0, 0, :2] = [1e-30, -0.0]
    cos, sin = _rope_tables(max_pos + new_len + 3, d)
    got = _run_append(compute, q, k, v, cos, sin, codes, scales, tables, positions, block_size, cache_dtype)
    assert got[3] is None
    where = positions[:, None] + np.arange(new_len)
    want_codes, want_scales = [c.copy() for c in codes], [s.copy() for s in scales]
    for x, c, s in ((_rotate32(k, cos[where][:, :, None], sin[where][:, :, None]), want_codes[0], want_scales[0]), (v, want_codes[1], want_scales[1])):
        assert not _append_reference(x, c, s, tables, positions, block_size, cache_dtype, cos.shape[0])
    _check_append(got, (want_codes, want_scales))  # pages and rows that the call does not own are part of the comparison
    if hq:
        assert np.array_equal(got[0].view(np.uint32), _rotate32(q, cos[where][:, :, None], sin[where][:, :, None]).view(np.uint32))


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [0, 1])
def test_appended_values_are_within_half_a_step(compute, cache_dtype):
    """Token by token into one page: each value ends within its roundings of what was written (one half step when it is
    coded, one more for each time its page's scale grew, all measured at the page's last scale)."""
    rng = np.random.default_rng(5)
    hkv, d, n = 2, 128, 16
    x = rng.standard_normal((n, hkv, d)).astype(np.float32) * np.linspace(0.2, 3, n, dtype=np.float32)[:, None, None]
    codes = [np.full((2 * 16, hkv, d), 0x11, np.uint8) for _ in range(2)]
    scales = [np.full((2, hkv), 9.0, np.float32) for _ in range(2)]
    cos, sin = np.ones((32, d // 2), np.float32), np.zeros((32, d // 2), np.float32)
    tables = np.array([[1]], np.int32)
    growth = np.zeros((n, hkv))
    for t in range(n):
        before = scales[0][1].copy() if t else np.zeros(hkv)
        _, codes, scales, err = _run_append(compute, None, x[None, t:t + 1], x[None, t:t + 1], cos, sin, codes, scales, tables,
                                            np.array([t], np.int32), 16, cache_dtype)
        assert err is None
        growth[t] += 1
        growth[:t] += scales[0][1] > before
    held = R.pool_values(codes[0], scales[0], cache_dtype, 16)[16:]
    step = scales[0][1][None, :, None] * (1.0 if cache_dtype == 0 else np.maximum(np.abs(held) / scales[0][1][None, :, None] / 8, 2.0 ** -9) * 1.1)
    # 2^-22: the divisions and products around the roundings
    assert (np.abs(held - x) <= 0.5 * step * growth[:, :, None] * (1.0 if cache_dtype == 0 else 1.15) + np.abs(x) * 2.0 ** -22).all()
    assert np.array_equal(codes[0], codes[1]) and (codes[0][:16] == 0x11).all()


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [0, 1])
def test_append_drops_and_reports_what_is_not_finite(compute, cache_dtype):
    from granite_b200.capi import ErrorCode
    rng = np.random.default_rng(6)
    hkv, d, batch, n = 2, 64, 2, 4
    k, v = (rng.standard_normal((batch, n, hkv, d), dtype=np.float32) for _ in range(2))
    v[0, 1, 0, 5], v[0, 2, 1, 6], v[1, 0, 0, 0] = np.nan, np.inf, -np.inf
    positions = np.array([2, 30], np.int32)
    tables, blocks = _table(rng, positions + n, 16)
    pools = [R.random_pool(rng, blocks, 16, hkv, d, cache_dtype) for _ in range(2)]
    codes, scales = [p[0] for p in pools], [p[1] for p in pools]
    cos, sin = _rope_tables(64, d)
    got = _run_append(compute, None, k, v, cos, sin, codes, scales, tables, positions, 16, cache_dtype)
    assert got[3] is not None and got[3].code == ErrorCode.InvalidArgument and "infinite" in str(got[3])
    where = positions[:, None] + np.arange(n)
    want_codes, want_scales = [c.copy() for c in codes], [s.copy() for s in scales]
    _append_reference(_rotate32(k, cos[where][:, :, None], sin[where][:, :, None]), want_codes[0], want_scales[0], tables, positions, 16, cache_dtype, 64)
    assert _append_reference(v, want_codes[1], want_scales[1], tables, positions, 16, cache_dtype, 64)
    _check_append(got, (want_codes, want_scales))


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [0, 1])
def test_append_skips_and_reports_what_cannot_be_placed(compute, cache_dtype):
    """A start before 0, an end beyond the RoPE table or the block table, a bad table entry: those tokens are left out, the others
    are written, and sync reports it; the next call is clean."""
    from granite_b200.capi import ErrorCode
    rng = np.random.default_rng(7)
    hkv, d, n = 2, 64, 20
    positions = np.array([-3, 50, 5, 1], np.int32)
    for bad in ("position", "entry"):
        tables = np.arange(16, dtype=np.int32).reshape(4, 4)
        pos = positions.copy() if bad == "position" else np.array([0, 3, 5, 1], np.int32)
        if bad == "entry":
            tables[1, 0], tables[2, 1] = -1, 16
        pools = [R.random_pool(rng, 16, 16, hkv, d, cache_dtype) for _ in range(2)]
        codes, scales = [p[0] for p in pools], [p[1] for p in pools]
        k, v = (rng.standard_normal((4, n, hkv, d), dtype=np.float32) for _ in range(2))
        q = rng.standard_normal((4, n, 4, d), dtype=np.float32)
        cos, sin = _rope_tables(60, d)
        got = _run_append(compute, q, k, v, cos, sin, codes, scales, tables, pos, 16, cache_dtype)
        assert got[3] is not None and got[3].code == ErrorCode.InvalidArgument
        where = pos[:, None] + np.arange(n)
        ok = ((where >= 0) & (where < 60))[:, :, None, None]
        at = np.clip(where, 0, 59)
        want_codes, want_scales = [c.copy() for c in codes], [s.copy() for s in scales]
        ref_tables = np.where(tables >= 16, -1, tables)
        _append_reference(_rotate32(k, cos[at][:, :, None], sin[at][:, :, None]), want_codes[0], want_scales[0], ref_tables, pos, 16, cache_dtype, 60)
        _append_reference(v, want_codes[1], want_scales[1], ref_tables, pos, 16, cache_dtype, 60)
        _check_append(got, (want_codes, want_scales))
        want_q = np.where(ok, _rotate32(q, cos[at][:, :, None], sin[at][:, :, None]), q)
        assert np.array_equal(got[0].view(np.uint32), want_q.view(np.uint32))
    compute.sync()


# --------------------------------------------------------------------------------------------- decode
def _decode_case(seed, lens, hq, hkv, d, cache_dtype, block_size=16, window=0, sinks=0, poison=True):
    rng = np.random.default_rng(seed)
    lens = np.asarray(lens, np.int32)
    tables, blocks = _table(rng, lens, block_size)
    (kc, ks), (vc, vs) = (R.random_pool(rng, blocks, block_size, hkv, d, cache_dtype) for _ in range(2))
    kc, vc, ks, vs = kc.copy(), vc.copy(), ks.copy(), vs.copy()
    q = rng.standard_normal((len(lens), hq, d), dtype=np.float32)
    scale = 1.0 / np.sqrt(d)
    kv, vv = R.pool_values(kc, ks, cache_dtype, block_size), R.pool_values(vc, vs, cache_dtype, block_size)
    want, bound = np.zeros((len(lens), hq, d)), np.zeros((len(lens), hq, 1))
    live = np.zeros(blocks * block_size, bool)
    for b, n in enumerate(lens):
        k, v = R.rows_of(kv, tables[b], n, block_size), R.rows_of(vv, tables[b], n, block_size)
        o, e = R.attend(q[b:b + 1].astype(np.float64), k, v, [n - 1], scale, window, sinks)
        want[b], bound[b] = o[0], e[0]
        seen = R.visible([n - 1], n, window, sinks)[0] if n else np.zeros(0, bool)
        for j in np.nonzero(seen)[0]:
            live[tables[b, j // block_size] * block_size + j % block_size] = True
        for pg in range((n + block_size - 1) // block_size):
            if not seen[pg * block_size:(pg + 1) * block_size].any():
                tables[b, pg] = -1 - pg  # a page that nothing sees may be freed
    if poison and cache_dtype == 1:  # masked rows hold NaN codes
        kc[~live], vc[~live] = 0x7F, 0xFF
    if poison:  # scales of pages without a live row are never used
        dead = ~live.reshape(blocks, block_size).any(1)
        ks[dead], vs[dead] = np.nan, np.inf
    return dict(q=q, kc=kc, vc=vc, ks=ks, vs=vs, tables=tables, lens=lens, blocks=blocks, scale=scale, want=want, bound=bound)


def _run_decode(compute, c, hq, hkv, d, cache_dtype, block_size=16, window=0, sinks=0):
    import torch
    out = torch.full(c["q"].shape, float("nan"), device=DEV)
    held = [_dev(c[n]) for n in ("q", "kc", "vc", "ks", "vs", "tables", "lens")]
    compute.batched_paged_attention_decode_q8(*held, out, len(c["lens"]), hq, hkv, d, block_size, c["tables"].shape[1], c["scale"],
                                              num_blocks=c["blocks"], cache_dtype=cache_dtype, window=window, sinks=sinks)
    compute.sync()
    return out.cpu().numpy()


SHAPES = [(32, 8, 128), (8, 8, 128), (16, 2, 128), (8, 1, 64), (12, 4, 64), (10, 2, 128), (16, 1, 128), (32, 1, 64), (24, 3, 128), (64, 16, 64),
          (6, 3, 40), (4, 2, 256), (24, 1, 96)]


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [0, 1])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_decode_q8_small_lengths(compute, cache_dtype, hq, hkv, d):
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 49, 100, 5, 0, 130]
    c = _decode_case(hq * 7 + d, lens, hq, hkv, d, cache_dtype)
    got = _run_decode(compute, c, hq, hkv, d, cache_dtype)
    R.assert_close(got, c["want"], c["bound"], what=f"{hq}/{hkv}/{d}")
    assert not got[0].any() and not got[14].any()


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [0, 1])
@pytest.mark.parametrize("hq,hkv,d,lens", [
    (32, 8, 128, [512]), (32, 8, 128, [2048]), (8, 2, 64, [2047, 1999]), (32, 8, 128, [6001]), (16, 4, 128, [9000, 33, 0, 4100]), (64, 8, 128, [1500, 800, 3111] * 14),
    (32, 8, 64, [700, 1300, 40] * 30), (8, 1, 128, [5000, 1, 77]), (16, 16, 128, [300] * 20), (16, 1, 128, [1234] * 50), (32, 8, 128, [90, 700, 5] * 100)])
def test_decode_q8_longer_batches(compute, cache_dtype, hq, hkv, d, lens):
    """One sequence and many, cut between CTAs and not, above and below 192 sequences."""
    c = _decode_case(len(lens) + d, lens, hq, hkv, d, cache_dtype)
    R.assert_close(_run_decode(compute, c, hq, hkv, d, cache_dtype), c["want"], c["bound"], what=f"{hq}/{hkv}/{d} {lens[:3]}")


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [0, 1])
@pytest.mark.parametrize("block_size", [1, 8, 32, 48])
def test_decode_q8_other_page_sizes(compute, cache_dtype, block_size):
    c = _decode_case(block_size, [1, 8, 33, 0, 100], 8, 2, 128, cache_dtype, block_size, window=40, sinks=3)
    R.assert_close(_run_decode(compute, c, 8, 2, 128, cache_dtype, block_size, 40, 3), c["want"], c["bound"])


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [0, 1])
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (8, 2, 64), (16, 1, 128), (6, 3, 40)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (17, 5), (64, 16), (100, 33), (100, 200), (4000, 4), (0x7fffffff, 0xffffffff)])
def test_decode_q8_windows(compute, cache_dtype, hq, hkv, d, window, sinks):
    lens = [0, 1, 15, 16, 17, 40, 116, 117, 118, 133, 300, 777]
    c = _decode_case(window % 1000 + sinks % 1000 + d, lens, hq, hkv, d, cache_dtype, window=window, sinks=sinks)
    R.assert_close(_run_decode(compute, c, hq, hkv, d, cache_dtype, 16, window, sinks), c["want"], c["bound"], what=f"{window} {sinks}")


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [0, 1])
def test_decode_q8_extreme_scales(compute, cache_dtype):
    """Pages of zeros (scale 0), V scales that grow and fall by 2^60 within a sequence."""
    hq, hkv, d, n = 8, 2, 128, 1000
    c = _decode_case(3, [n, 64], hq, hkv, d, cache_dtype, poison=False)
    rng = np.random.default_rng(4)
    c["vs"] = (c["vs"] * 2.0 ** rng.integers(-30, 31, c["vs"].shape)).astype(np.float32)
    for i in (3, 17):
        page = c["tables"][0, i]
        c["ks"][page], c["vs"][page] = 0, 0
        c["kc"][page * 16:page * 16 + 16] = 0
        c["vc"][page * 16:page * 16 + 16] = 0
    kv, vv = R.pool_values(c["kc"], c["ks"], cache_dtype, 16), R.pool_values(c["vc"], c["vs"], cache_dtype, 16)
    got = _run_decode(compute, c, hq, hkv, d, cache_dtype)
    for b, m in enumerate(c["lens"]):
        o, e = R.attend(c["q"][b:b + 1].astype(np.float64), R.rows_of(kv, c["tables"][b], m, 16), R.rows_of(vv, c["tables"][b], m, 16), [m - 1], c["scale"])
        R.assert_close(got[b], o[0], e[0], what=f"sequence {b}")


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [0, 1])
def test_decode_q8_queries_out_of_the_ordinary(compute, cache_dtype):
    """Queries of zeros and of very small and large magnitude come out right, a NaN or infinity stays in its own head."""
    hq, hkv, d = 8, 2, 128
    c = _decode_case(70, [100, 333], hq, hkv, d, cache_dtype)
    q = c["q"].copy()
    q[0, 0], q[0, 1], q[0, 2] = 0, q[0, 1] * 1e-25, q[0, 2] * 8
    q[1, 3, 7], q[1, 5, 0] = np.nan, np.inf
    kv, vv = R.pool_values(c["kc"], c["ks"], cache_dtype, 16), R.pool_values(c["vc"], c["vs"], cache_dtype, 16)
    got = _run_decode(compute, dict(c, q=q), hq, hkv, d, cache_dtype)
    assert np.isnan(got[1, 3]).all() and not np.isfinite(got[1, 5]).any()
    for b, n in enumerate(c["lens"]):
        fine = [h for h in range(hq) if np.isfinite(q[b, h]).all()]
        finite = np.where(np.isfinite(q[b:b + 1]), q[b:b + 1], 0).astype(np.float64)
        o, e = R.attend(finite, R.rows_of(kv, c["tables"][b], n, 16), R.rows_of(vv, c["tables"][b], n, 16), [n - 1], c["scale"])
        R.assert_close(got[b][fine], o[0][fine], e[0][fine], what=f"sequence {b}")


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [0, 1])
def test_decode_q8_reports_bad_tables_and_lengths(compute, cache_dtype):
    """Entries outside the pool and lengths outside the table are reported, not followed; the other sequences come out right."""
    from granite_b200.capi import ErrorCode, GraniteCudaError
    c = _decode_case(9, [100, 50, 300], 8, 2, 128, cache_dtype)
    for what, value in (("tables", c["blocks"]), ("tables", -1), ("lens", -1), ("lens", c["tables"].shape[1] * 16 + 1)):
        bad = dict(c)
        bad[what] = c[what].copy()
        if what == "tables":
            bad[what][1, 2] = value
        else:
            bad[what][1] = value
        with pytest.raises(GraniteCudaError) as e:
            _run_decode(compute, bad, 8, 2, 128, cache_dtype)
        assert e.value.code == ErrorCode.InvalidArgument
    R.assert_close(_run_decode(compute, c, 8, 2, 128, cache_dtype), c["want"], c["bound"])


# --------------------------------------------------------------------------------------------- prefill
def _prefill_case(seed, seq, start, hq, hkv, d, cache_dtype, half, block_size=16, window=0, sinks=0):
    rng = np.random.default_rng(seed)
    n = start + seq
    tables, blocks = _table(rng, [n], block_size)
    (kc, ks), (vc, vs) = (R.random_pool(rng, blocks, block_size, hkv, d, cache_dtype) for _ in range(2))
    kc, vc, ks, vs = kc.copy(), vc.copy(), ks.copy(), vs.copy()
    q = rng.standard_normal((seq, hq, d), dtype=np.float32)
    if half:
        q = q.astype(np.float16).astype(np.float32)
    scale = 1.0 / np.sqrt(d)
    k = R.rows_of(R.pool_values(kc, ks, cache_dtype, block_size), tables[0], n, block_size)
    v = R.rows_of(R.pool_values(vc, vs, cache_dtype, block_size), tables[0], n, block_size)
    want, bound = R.attend(q.astype(np.float64), k, v, start + np.arange(seq), scale, window, sinks)
    seen = R.visible(start + np.arange(seq), n, window, sinks).any(0)
    live = np.zeros(blocks * block_size, bool)
    for j in np.nonzero(seen)[0]:
        live[tables[0, j // block_size] * block_size + j % block_size] = True
    for pg in range(tables.shape[1]):
        if not seen[pg * block_size:(pg + 1) * block_size].any():
            tables[0, pg] = blocks + 7
    if cache_dtype == 1:
        kc[~live], vc[~live] = 0x7F, 0xFF
    dead = ~live.reshape(blocks, block_size).any(1)
    ks[dead], vs[dead] = np.inf, np.nan
    return dict(q=q, kc=kc, vc=vc, ks=ks, vs=vs, tables=tables, blocks=blocks, scale=scale, want=want, bound=bound)


def _run_prefill(compute, c, start, hkv, cache_dtype, half, block_size=16, window=0, sinks=0):
    import torch
    seq, hq, d = c["q"].shape
    dt = torch.float16 if half else torch.float32
    out = torch.full((seq, hq, d), float("nan"), device=DEV, dtype=dt)
    held = [_dev(c["q"], dt)] + [_dev(c[n]) for n in ("kc", "vc", "ks", "vs", "tables")]
    compute.paged_prefill_attention_q8(*held, out, hq, hkv, seq, start, d, block_size, c["tables"].shape[1], c["blocks"], c["scale"],
                                       cache_dtype, q_dtype=int(half), out_dtype=int(half), window=window, sinks=sinks)
    compute.sync()
    return out.float().cpu().numpy()


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [0, 1])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("seq,start,hq,hkv,d", [(1, 0, 8, 2, 128), (1, 300, 8, 2, 128), (2, 14, 8, 8, 64), (127, 1, 4, 1, 128), (128, 0, 8, 2, 128),
                                                (129, 127, 8, 2, 64), (300, 333, 6, 3, 128), (40, 1000, 32, 8, 128), (17, 5, 4, 2, 40)])
def test_prefill_q8(compute, cache_dtype, half, seq, start, hq, hkv, d):
    c = _prefill_case(seq + start, seq, start, hq, hkv, d, cache_dtype, half)
    R.assert_close(_run_prefill(compute, c, start, hkv, cache_dtype, half), c["want"], c["bound"], half, f"{seq}@{start}")


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [0, 1])
@pytest.mark.parametrize("window,sinks", [(1, 0), (30, 7), (128, 0), (129, 130), (500, 4)])
@pytest.mark.parametrize("seq,start,d,block_size", [(150, 0, 128, 16), (200, 555, 128, 16), (130, 300, 64, 16), (60, 100, 128, 32)])
def test_prefill_q8_windows(compute, cache_dtype, window, sinks, seq, start, d, block_size):
    c = _prefill_case(seq + window, seq, start, 4, 2, d, cache_dtype, False, block_size, window, sinks)
    got = _run_prefill(compute, c, start, 2, cache_dtype, False, block_size, window, sinks)
    R.assert_close(got, c["want"], c["bound"], what=f"{seq}@{start} {window}+{sinks}")


# --------------------------------------------------------------------------------------------- together
@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [0, 1])
def test_prompt_then_steps_over_the_8bit_cache(compute, cache_dtype):
    """A prompt enters in two chunks (append, then attention over the cache), then single tokens follow: every output is the
    attention over the values that the cache then holds."""
    import torch
    rng = np.random.default_rng(11)
    hq, hkv, d, n = 8, 2, 128, 100
    tables = rng.permutation(8).astype(np.int32)[None]
    cos, sin = _rope_tables(128, d)
    kc, vc = (torch.zeros((128, hkv, d), dtype=torch.uint8, device=DEV) for _ in range(2))
    ks, vs = (torch.zeros((8, hkv), device=DEV) for _ in range(2))
    td, cd, sd = _dev(tables), _dev(cos), _dev(sin)
    at = 0
    for step in (60, 37, 1, 1, 1):
        q, k, v = (torch.from_numpy(rng.standard_normal((1, step, h, d), dtype=np.float32)).to(DEV) for h in (hq, hkv, hkv))
        pos = torch.tensor([at], dtype=torch.int32, device=DEV)
        q_in, k_in, v_in = (t.cpu().numpy() for t in (q, k, v))
        compute.rope_paged_kv_cache_append_q8(q, k, v, cd, sd, kc, vc, ks, vs, td, pos, 1, step, hq, hkv, d, 16, 8, 8, 128, cache_dtype)
        out = torch.full((step, hq, d), float("nan"), device=DEV)
        if step > 1:
            compute.paged_prefill_attention_q8(q, kc, vc, ks, vs, td, out, hq, hkv, step, at, d, 16, 8, 8, 1 / np.sqrt(d), cache_dtype)
        else:
            compute.batched_paged_attention_decode_q8(q, kc, vc, ks, vs, td, pos + 1, out, 1, hq, hkv, d, 16, 8, 1 / np.sqrt(d),
                                                      num_blocks=8, cache_dtype=cache_dtype)
        compute.sync()
        at += step
        values = [R.rows_of(R.pool_values(c.cpu().numpy(), s.cpu().numpy(), cache_dtype, 16), tables[0], at, 16) for c, s in ((kc, ks), (vc, vs))]
        where = np.arange(at - step, at)
        rotated = _rotate32(q_in, cos[where][None, :, None], sin[where][None, :, None])
        assert np.array_equal(q.cpu().numpy(), rotated)
        want, bound = R.attend(rotated[0].astype(np.float64), *values, where, 1 / np.sqrt(d))
        R.assert_close(out.cpu().numpy(), want, bound, what=f"{step} tokens at {at - step}")
        # what the cache holds is what was written, to 8 bits: half a step of each page's scale, twice over for growth
        for i, (x, s) in enumerate(((_rotate32(k_in, cos[where][None, :, None], sin[where][None, :, None]), ks), (v_in, vs))):
            sc = s.cpu().numpy()[tables[0, where // 16]][:, :, None]
            err = np.abs(values[i][at - step:] - x[0])
            assert (err <= (0.5 * sc if cache_dtype == 0 else np.maximum(np.abs(x[0]) * 2.0 ** -4, sc * 2.0 ** -10)) * 1.0001).all()


@pytest.mark.gpu
def test_q8_calls_replay_from_a_graph_on_another_stream():
    import torch
    import granite_b200 as g
    side = torch.cuda.Stream(device=DEV)
    objs = [g.CudaCompute(0, side.cuda_stream), g.CudaCompute(0)]
    hq, hkv, d = 32, 8, 128
    cases = [_decode_case(20, [700, 30, 0, 2000, 9], hq, hkv, d, 0), _decode_case(21, [1500], hq, hkv, d, 1, window=300, sinks=4),
             _decode_case(22, [400, 500] * 25, hq, hkv, d, 1)]
    held = [[_dev(c[n]) for n in ("q", "kc", "vc", "ks", "vs", "tables", "lens")] for c in cases]
    outs = [torch.zeros(c["q"].shape, device=DEV) for c in cases]
    p = _prefill_case(23, 70, 90, hq, hkv, d, 0, False)
    p_held = [_dev(p["q"])] + [_dev(p[n]) for n in ("kc", "vc", "ks", "vs", "tables")]
    p_out = torch.zeros(p["q"].shape, device=DEV)

    def calls(o):
        for c, h, out, (dt, w, s) in zip(cases, held, outs, ((0, 0, 0), (1, 300, 4), (1, 0, 0))):
            o.batched_paged_attention_decode_q8(*h, out, len(c["lens"]), hq, hkv, d, 16, c["tables"].shape[1], c["scale"],
                                                num_blocks=c["blocks"], cache_dtype=dt, window=w, sinks=s)
        o.paged_prefill_attention_q8(*p_held, p_out, hq, hkv, 70, 90, d, 16, p["tables"].shape[1], p["blocks"], p["scale"], 0)

    torch.cuda.synchronize()
    for o in objs:
        calls(o)
        o.sync()
    for t in outs + [p_out]:
        t.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        calls(objs[0])
    torch.cuda.synchronize()
    assert not outs[0].any()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    objs[0].sync()
    for c, out in zip(cases, outs):
        R.assert_close(out.cpu().numpy(), c["want"], c["bound"], what="replay")
    R.assert_close(p_out.cpu().numpy(), p["want"], p["bound"], what="prefill replay")
    del graph
    for o in objs:
        o.shutdown()


@pytest.mark.gpu
def test_a_captured_graph_outlives_the_growth_of_the_workspace():
    """A graph holds the workspace that it was captured with; a later, larger call must not take it away."""
    import torch
    import granite_b200 as g
    side = torch.cuda.Stream(device=DEV)
    o = g.CudaCompute(0, side.cuda_stream)
    hq, hkv, d = 32, 8, 128
    c = _decode_case(30, [900, 1200, 40] * 20, hq, hkv, d, 0)
    held = [_dev(c[n]) for n in ("q", "kc", "vc", "ks", "vs", "tables", "lens")]
    out = torch.zeros(c["q"].shape, device=DEV)

    def step():
        o.batched_paged_attention_decode_q8(*held, out, len(c["lens"]), hq, hkv, d, 16, c["tables"].shape[1], c["scale"], num_blocks=c["blocks"], cache_dtype=0)

    torch.cuda.synchronize()
    step()
    o.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    p = _prefill_case(31, 300, 2000, 8, 2, d, 1, False)  # more workspace than the step's
    big = _decode_case(32, [20] * 400, hq, hkv, d, 0)     # more sequences: larger counters and tables
    p_out, b_out = torch.zeros(p["q"].shape, device=DEV), torch.zeros(big["q"].shape, device=DEV)
    p_held = [_dev(p["q"])] + [_dev(p[n]) for n in ("kc", "vc", "ks", "vs", "tables")]
    b_held = [_dev(big[n]) for n in ("q", "kc", "vc", "ks", "vs", "tables", "lens")]
    torch.cuda.synchronize()
    o.paged_prefill_attention_q8(*p_held, p_out, 8, 2, 300, 2000, d, 16, p["tables"].shape[1], p["blocks"], p["scale"], 1)
    o.batched_paged_attention_decode_q8(*b_held, b_out, 400, hq, hkv, d, 16, big["tables"].shape[1], big["scale"], num_blocks=big["blocks"], cache_dtype=0)
    o.sync()
    junk = [torch.full((1 << 22,), float("nan"), device=DEV) for _ in range(8)]  # whatever memory was given back is written over
    out.zero_()
    torch.cuda.synchronize()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    o.sync()
    R.assert_close(out.cpu().numpy(), c["want"], c["bound"], what="replay after growth")
    R.assert_close(p_out.cpu().numpy(), p["want"], p["bound"], what="prefill")
    R.assert_close(b_out.cpu().numpy(), big["want"], big["bound"], what="large batch")
    del graph, junk
    o.shutdown()


@pytest.mark.gpu
def test_two_objects_work_at_the_same_time():
    """Two compute objects on two streams, 8-bit decode and prefill interleaved: no shared workspace, counters or status."""
    import torch
    import granite_b200 as g
    streams = [torch.cuda.Stream(device=DEV) for _ in range(2)]
    objs = [g.CudaCompute(0, s.cuda_stream) for s in streams]
    hq, hkv, d = 16, 4, 128
    cs = [_decode_case(40 + i, [700, 1500, 33] * 15, hq, hkv, d, i) for i in range(2)]
    ps = [_prefill_case(50 + i, 90, 1000, hq, hkv, d, i, False) for i in range(2)]
    held = [[_dev(c[n]) for n in ("q", "kc", "vc", "ks", "vs", "tables", "lens")] for c in cs]
    p_held = [[_dev(p["q"])] + [_dev(p[n]) for n in ("kc", "vc", "ks", "vs", "tables")] for p in ps]
    outs, p_outs = [torch.zeros(c["q"].shape, device=DEV) for c in cs], [torch.zeros(p["q"].shape, device=DEV) for p in ps]
    torch.cuda.synchronize()
    for _ in range(6):
        for i, o in enumerate(objs):
            o.batched_paged_attention_decode_q8(*held[i], outs[i], 45, hq, hkv, d, 16, cs[i]["tables"].shape[1], cs[i]["scale"], num_blocks=cs[i]["blocks"], cache_dtype=i)
            o.paged_prefill_attention_q8(*p_held[i], p_outs[i], hq, hkv, 90, 1000, d, 16, ps[i]["tables"].shape[1], ps[i]["blocks"], ps[i]["scale"], i)
    for i, o in enumerate(objs):
        o.sync()
        R.assert_close(outs[i].cpu().numpy(), cs[i]["want"], cs[i]["bound"], what=f"decode {i}")
        R.assert_close(p_outs[i].cpu().numpy(), ps[i]["want"], ps[i]["bound"], what=f"prefill {i}")
        o.shutdown()


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [0, 1])
def test_split_pages_give_the_same_bits_every_time(compute, cache_dtype):
    """1, 2 and 4 KV heads share a head's pages among warps: many runs of the same call, long enough to wrap the ring, agree."""
    import torch
    for hq, hkv, d in ((16, 4, 128), (8, 2, 128), (4, 1, 128), (16, 4, 64), (4, 1, 64)):
        c = _decode_case(60 + hkv + d, [3000, 2000, 1000, 17] * 12, hq, hkv, d, cache_dtype)
        held = [_dev(c[n]) for n in ("q", "kc", "vc", "ks", "vs", "tables", "lens")]
        outs = []
        for _ in range(40):
            out = torch.empty(c["q"].shape, device=DEV)
            compute.batched_paged_attention_decode_q8(*held, out, len(c["lens"]), hq, hkv, d, 16, c["tables"].shape[1], c["scale"], num_blocks=c["blocks"], cache_dtype=cache_dtype)
            outs.append(out)
        compute.sync()
        R.assert_close(outs[0].cpu().numpy(), c["want"], c["bound"], what=f"{hq}/{hkv}/{d}")
        assert all(torch.equal(outs[0], o) for o in outs[1:])


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype,half,seq,start,window", [(0, False, 10, 9000, 0), (1, True, 300, 5000, 0), (0, False, 140, 7000, 6000), (1, False, 1, 4097, 0)])
def test_prefill_q8_cut_along_the_keys(compute, cache_dtype, half, seq, start, window):
    """Few queries over many keys, and more key tiles than one accumulator takes: chunks and their merge."""
    c = _prefill_case(seq + start, seq, start, 4, 2, 128, cache_dtype, half, window=window, sinks=3 if window else 0)
    got = _run_prefill(compute, c, start, 2, cache_dtype, half, window=window, sinks=3 if window else 0)
    R.assert_close(got, c["want"], c["bound"], half, f"{seq}@{start}")


# --------------------------------------------------------------------------------------------- refusals (no device needed)
def _refusal(fn, *args):
    from granite_b200 import capi
    code = fn(None, *args)
    assert code != 0
    return capi.ErrorCode(code), capi.last_error()


def _append_args(**kw):
    from granite_b200 import capi
    a = dict(q=256, k=256, v=256, cos_table=256, sin_table=256, k_cache=256, v_cache=256, block_tables=256, positions=256, batch_size=1, new_len=1,
             num_heads=4, num_kv_heads=2, head_dim=128, block_size=16, max_blocks_per_seq=4, num_blocks=4, table_len=64)
    a.update({k: v for k, v in kw.items() if k in a})
    x = dict(k_scales=256, v_scales=256, cache_dtype=0)
    x.update({k: v for k, v in kw.items() if k in x})
    return C.byref(capi.RopeAppendArgs(**a)), C.byref(capi.Q8Cache(**x))


@pytest.mark.parametrize("kw,code,word", [
    (dict(k=None), "NullPointer", "null"), (dict(k_scales=None), "NullPointer", "null"), (dict(cache_dtype=2), "InvalidArgument", "cache_dtype"),
    (dict(head_dim=12), "InvalidArgument", "head_dim"), (dict(head_dim=264), "InvalidArgument", "head_dim"), (dict(head_dim=0), "InvalidArgument", "head_dim"),
    (dict(num_kv_heads=0), "InvalidArgument", "empty"), (dict(block_size=0), "InvalidArgument", "empty"), (dict(num_blocks=0), "InvalidArgument", "empty"),
    (dict(num_heads=0), "InvalidArgument", "empty"), (dict(k_cache=264), "InvalidArgument", "aligned"), (dict(v=260), "InvalidArgument", "aligned"),
    (dict(cos_table=260), "InvalidArgument", "aligned"), (dict(batch_size=1 << 31), "InvalidArgument", "range"), (dict(), "NullPointer", "compute object")])
def test_append_q8_refusals(kw, code, word):
    from granite_b200 import capi
    got, text = _refusal(capi.lib.granite_cuda_rope_paged_kv_cache_append_q8, *_append_args(**kw))
    assert got.name == code and word in text


def _decode_args(**kw):
    from granite_b200 import capi
    a = dict(q=256, k_cache=256, v_cache=256, block_tables=256, seq_lens=256, output=256, batch_size=1, num_heads=4, num_kv_heads=2, head_dim=128,
             block_size=16, max_blocks_per_seq=4, num_blocks=4, scale=0.1)
    a.update({k: v for k, v in kw.items() if k in a})
    x = dict(k_scales=256, v_scales=256, cache_dtype=0)
    x.update({k: v for k, v in kw.items() if k in x})
    w = C.byref(capi.AttentionWindow(kw["window"], 0)) if "window" in kw else None
    return C.byref(capi.PagedDecodeArgs(**a)), C.byref(capi.Q8Cache(**x)), w


VIEW_REFUSALS = [(dict(k_cache=None), "NullPointer", "null"), (dict(q=None), "NullPointer", "null"), (dict(v_scales=None), "NullPointer", "scales"),
                 (dict(cache_dtype=7), "InvalidArgument", "cache_dtype"), (dict(window=0), "InvalidArgument", "window"),
                 (dict(num_heads=5), "InvalidArgument", "multiple"), (dict(num_heads=0), "InvalidArgument", "multiple"), (dict(num_kv_heads=0), "InvalidArgument", "multiple"),
                 (dict(head_dim=100), "InvalidArgument", "head_dim"), (dict(head_dim=512), "InvalidArgument", "head_dim"), (dict(k_cache=264), "InvalidArgument", "aligned"),
                 (dict(q=264), "InvalidArgument", "aligned"), (dict(num_blocks=0), "InvalidArgument", "empty"), (dict(block_size=0), "InvalidArgument", "empty"),
                 (dict(max_blocks_per_seq=1 << 28), "InvalidArgument", "2^31"), (dict(scale=-0.1), "InvalidArgument", "scale"), (dict(scale=0.0), "InvalidArgument", "scale"),
                 (dict(scale=float("nan")), "InvalidArgument", "scale"), (dict(scale=float("inf")), "InvalidArgument", "scale"), (dict(), "NullPointer", "compute object")]


@pytest.mark.parametrize("kw,code,word", VIEW_REFUSALS)
def test_decode_q8_refusals(kw, code, word):
    from granite_b200 import capi
    got, text = _refusal(capi.lib.granite_cuda_batched_paged_attention_decode_q8, *_decode_args(**kw))
    assert got.name == code and word in text


@pytest.mark.parametrize("kw,code,word", VIEW_REFUSALS + [(dict(start_pos=60, seq_q=5), "InvalidArgument", "beyond"), (dict(q_dtype=2), "InvalidArgument", "dtype")])
def test_prefill_q8_refusals(kw, code, word):
    from granite_b200 import capi
    a = dict(q=256, k_cache=256, v_cache=256, block_table=256, output=256, num_heads=4, num_kv_heads=2, seq_q=4, start_pos=0, head_dim=128, block_size=16,
             max_blocks_per_seq=4, num_blocks=4, scale=0.1)
    a.update({k: v for k, v in kw.items() if k in a or k == "q_dtype"})
    _, x, w = _decode_args(**kw)
    got, text = _refusal(capi.lib.granite_cuda_paged_prefill_attention_q8, C.byref(capi.PagedPrefillArgs(**a)), x, w)
    assert got.name == code and word in text


def test_structures_match_the_header(tmp_path):
    """GraniteCudaQ8Cache and GraniteCudaAttentionWindow as a C compiler lays them out, against the binding's."""
    import shutil
    import subprocess
    from pathlib import Path
    from granite_b200 import capi
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "granite_cuda.h"', "int main(void) {"]
    pairs = {"GraniteCudaQ8Cache": capi.Q8Cache, "GraniteCudaAttentionWindow": capi.AttentionWindow}
    for name, cls in pairs.items():
        lines.append(f'  printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    include = Path(__file__).resolve().parent.parent / "include"
    subprocess.run([cc, "-std=c11", f"-I{include}", str(src), "-o", str(exe)], check=True)
    out = dict(x.split() for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    for name, cls in pairs.items():
        assert int(out[name]) == C.sizeof(cls)
        for f, _ in cls._fields_:
            assert int(out[f"{name}.{f}"]) == getattr(cls, f).offset


def test_reference_encoding_is_the_format():
    """The tests' own e4m3 rounding, on every value, every midpoint and beyond the range; torch's cast as a second opinion."""
    import torch
    v = R.e4m3_values()
    fine = np.isfinite(v)
    assert np.array_equal(R.decode_codes(R.encode(v[fine], 1), 1), v[fine])
    grid = np.concatenate([np.linspace(-450, 450, 9001), 2.0 ** -np.arange(0, 14.0, 0.125), [0.0, -0.0]])
    mid = (v[:126] + v[1:127]) / 2
    x = np.concatenate([grid, mid, -mid]).astype(np.float32)
    x = x[np.abs(x) <= 448]
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(R.encode(x.astype(np.float64), 1), want)


def test_window_span_leaves_the_visible_keys():
    """The two ranges that the kernels walk ([0, min(sinks, lo)) and [lo, pos]) are the visible keys of the definition."""
    for window in (1, 2, 5, 16, 100):
        for sinks in (0, 1, 7, 40):
            for pos in range(0, 60):
                lo = pos - window + 1 if pos >= window else 0
                keys = sorted(set(range(min(sinks, lo))) | set(range(lo, pos + 1)))
                assert np.array_equal(np.nonzero(R.visible([pos], pos + 1, window, sinks)[0])[0], keys)
