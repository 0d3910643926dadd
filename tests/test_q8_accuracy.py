"""How exact attention over the 8-bit cache stays where magnitudes are spread: V scales that differ by many powers of two
between pages, with the weight on the pages of small values or with the large ones closed to a row, and small queries
against large keys.  Errors are held to each output's own sum of weight * |value|, not to the largest value of the call."""
import numpy as np
import pytest

import view_reference as R
from test_q8_cache import _dev, _table

DEV = "cuda:0"


def weighted_reference(q, codes, scales, v_codes, v_scales, pos, scale, cache_dtype, table, block_size=16, window=0, sinks=0):
    """64-bit attention of q [R, Hq, D] at positions pos, and the bound on the error of each output.  With w the weights (largest
    1), W their sum and A = sum w |v| / W:
      * a weight is off by (D + 8) 2^-24 S (its fp32 score, S = sum |q k| scale; Q as fp16 hi + lo under a power of two is within
        2^-22 of a head's largest element and counts there), by 2^-21 (exponential, hi + lo form), and by 2^-24 of the base-2 logarithms
        of the V scales' ratio and of the score, which are added in fp32: relative errors, each at most twice into the mean;
      * sums over n keys add n 2^-23 of A;
      * a product of weight and V scale is held as fp16 hi + lo, to 2^-25 where it is small, in units in which the row's largest
        product is at least 1/4: 2^-23 qmax max(w vs) / W for each key.
    The third result bounds the norm of a (row, head)'s errors: those of sums of at most 2^15 terms add up like a random walk, 2^-16.5
    of the norm of A; an error of a score moves all of a row alike and does not, so it counts in full: with s = sum |q k| scale of
    a key, D / 16 truncated steps of 2^-23 s at most, 2^-22 s for Q's form, and 2^-24 s for each of the products with
    scale and page scale and the subtraction of the maximum (in base-2 units, at most twice that): (D / 16 + 6) 2^-23 s, into
    the mean once by the weights and once by their sum."""
    rows, hq, d = q.shape
    n = int(max(pos)) + 1
    kv, vv = (R.rows_of(R.pool_values(c, s, cache_dtype, block_size), table, n, block_size) for c, s in ((codes, scales), (v_codes, v_scales)))
    at = table[np.arange(n) // block_size]
    seen = R.visible(pos, n, window, sinks)
    want, bound, norm = np.zeros((rows, hq, d)), np.zeros((rows, hq, d)), np.zeros((rows, hq))
    for h in range(hq):
        g = h // (hq // kv.shape[1])
        x = np.where(seen, (q[:, h] @ kv[:, g].T) * scale, -np.inf)
        big = np.where(seen, (np.abs(q[:, h]).max(1, keepdims=True) * np.abs(kv[:, g]).sum(1)[None]) * scale, 0).max(1, keepdims=True)
        top = x.max(1, keepdims=True)
        w = np.exp(x - top)
        total = w.sum(1, keepdims=True)
        vs = v_scales[at, g].astype(np.float64)
        live = vs[np.any(seen & (w > 0), 0)]
        spread = np.log2(live.max() / live[live > 0].min()) if (live > 0).any() else 0.0
        want[:, h] = w @ vv[:, g] / total
        mean = w @ np.abs(vv[:, g]) / total
        ws = w * ((np.abs(q[:, h]) @ np.abs(kv[:, g]).T) * scale)
        moved = ws @ np.abs(vv[:, g]) / total + ws.sum(1, keepdims=True) / total * mean
        norm[:, h] = 2.0 ** -16.5 * np.linalg.norm(mean, axis=-1) + (d / 16 + 6) * 2.0 ** -23 * np.linalg.norm(moved, axis=-1)
        rel = (d + 8) * 2.0 ** -24 * big + 2.0 ** -21 + 2.0 ** -24 * (spread + np.abs(top) * 1.443)
        floor = n * 2.0 ** -23 * R.QMAX[cache_dtype] * (w * vs[None]).max(1, keepdims=True) / total
        bound[:, h] = (2 * rel + n * 2.0 ** -23) * mean + floor
    return want, bound, norm


def check(got, want, bound, norm, what):
    got = np.asarray(got, np.float64)
    assert np.isfinite(got).all(), what
    over = np.abs(got - want) - bound
    assert over.max() <= 0, f"{what}: off by {np.abs(got - want).max():.3e}, {over.max():.3e} over the bound"
    off = np.linalg.norm(got - want, axis=-1) / norm
    assert off.max() <= 1, f"{what}: {off.max():.3g} times the bound on a row's norm at {np.unravel_index(off.argmax(), off.shape)}"


def spread_pools(rng, blocks, hkv, d, cache_dtype, table, n, q_dir, scale, v_log2, tilt):
    """Pools whose page scales of V are 2^v_log2[page] and whose keys give a token of logical page p the score
    -tilt * ln(V scale) + noise against q_dir [Hkv, D]: with tilt above 1 the weight sits on the pages of small values."""
    kc = np.zeros((blocks * 16, hkv, d), np.uint8)
    ks = np.ones((blocks, hkv), np.float32)
    vc, vs = R.random_pool(rng, blocks, 16, hkv, d, cache_dtype)
    vc, vs = vc.copy(), vs.copy()
    for p in range((n + 15) // 16):
        e = table[p]
        vs[e] = (vs[e] * 2.0 ** v_log2[p]).astype(np.float32)
        target = -tilt * np.log(vs[e].astype(np.float64))[None, :] + rng.standard_normal((16, hkv))
        k = target[..., None] * q_dir / ((q_dir ** 2).sum(-1, keepdims=True) * scale) + 0.05 * rng.standard_normal((16, hkv, d))
        ks[e] = (np.abs(k).max((0, 2)) / R.QMAX[cache_dtype]).astype(np.float32)
        kc[e * 16:e * 16 + 16] = R.encode(k / ks[e][None, :, None], cache_dtype)
    return kc, ks, vc, vs


PREFILLS = [(300, 0, 8, 2, 128), (140, 333, 4, 1, 64), (40, 1200, 4, 2, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [0, 1])
@pytest.mark.parametrize("seq,start,hq,hkv,d", PREFILLS)
@pytest.mark.parametrize("bits,tilt,order", [(12, 0.0, "later"), (24, 0.0, "later"), (40, 0.0, "later"), (20, 1.5, "mixed"), (30, 1.2, "earlier")])
def test_prefill_q8_with_spread_v_scales(compute, cache_dtype, seq, start, hq, hkv, d, bits, tilt, order):
    """`later`: V grows by 2^bits towards the chunk's end, so that early rows may not see the large pages; otherwise the weight sits
    on pages of small values."""
    import torch
    rng = np.random.default_rng(bits + seq + d)
    n, scale = start + seq, d ** -0.5
    tables, blocks = _table(rng, [n], 16)
    pages = (n + 15) // 16
    v_log2 = np.linspace(-bits, 0, pages)
    if order == "earlier":
        v_log2 = v_log2[::-1]
    if order == "mixed":
        v_log2 = rng.permutation(v_log2)
    q_dir = rng.standard_normal((hkv, d))
    q = (np.repeat(q_dir, hq // hkv, 0)[None] * (1 + 0.02 * rng.standard_normal((seq, hq, 1)))).astype(np.float32)
    kc, ks, vc, vs = spread_pools(rng, blocks, hkv, d, cache_dtype, tables[0], n, q_dir, scale, v_log2, tilt)
    ref = weighted_reference(q.astype(np.float64), kc, ks, vc, vs, start + np.arange(seq), scale, cache_dtype, tables[0])
    out = torch.full(q.shape, float("nan"), device=DEV)
    compute.paged_prefill_attention_q8(*[_dev(x) for x in (q, kc, vc, ks, vs, tables)], out, hq, hkv, seq, start, d, 16, tables.shape[1], blocks, scale, cache_dtype)
    compute.sync()
    check(out.cpu().numpy(), *ref, f"{seq}@{start} 2^{bits} {order}")


DECODES = [(8, 2, 128, [1000, 64, 333, 17]), (32, 8, 128, [2100, 700] * 12), (8, 1, 64, [900, 40]), (16, 2, 128, [3000, 500] * 40), (10, 2, 128, [777, 50]), (24, 2, 64, [600] * 3),
           (12, 1, 128, [500])]


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [0, 1])
@pytest.mark.parametrize("hq,hkv,d,lens", DECODES)
@pytest.mark.parametrize("bits,tilt", [(12, 1.3), (20, 1.5), (30, 1.2), (60, 1.4)])
def test_decode_q8_with_spread_v_scales(compute, cache_dtype, hq, hkv, d, lens, bits, tilt):
    """The weight sits on pages of small values, pages of large values have next to none: one sequence and many, cut between
    CTAs and warps and not."""
    import torch
    rng = np.random.default_rng(bits + hq + d)
    scale = d ** -0.5
    lens = np.asarray(lens, np.int32)
    kinds = {}  # sequences of one length share their pages, so that the reference is worked out once for each
    parts, tables, blocks = [], np.full((len(lens), (lens.max() + 15) // 16), -1, np.int32), 0
    q_dir = rng.standard_normal((hkv, d))
    q1 = (np.repeat(q_dir, hq // hkv, 0) * (1 + 0.02 * rng.standard_normal((hq, 1)))).astype(np.float32)
    for b, n in enumerate(lens):
        if n not in kinds:
            t, count = _table(rng, [n], 16)
            pages = (n + 15) // 16
            pools = spread_pools(rng, count, hkv, d, cache_dtype, t[0], n, q_dir, scale, rng.uniform(-bits, 0, pages), tilt)
            kinds[n] = (blocks, t[0], weighted_reference(q1[None].astype(np.float64), *pools, [n - 1], scale, cache_dtype, t[0]))
            parts.append(pools)
            blocks += count
        base, t, _ = kinds[n]
        tables[b, :len(t)] = t + base
    kc, ks, vc, vs = (np.concatenate(x) for x in zip(*parts))
    q = np.broadcast_to(q1, (len(lens), hq, d)).copy()
    out = torch.full(q.shape, float("nan"), device=DEV)
    compute.batched_paged_attention_decode_q8(*[_dev(x) for x in (q, kc, vc, ks, vs, tables, lens)], out, len(lens), hq, hkv, d, 16, tables.shape[1], scale,
                                              num_blocks=blocks, cache_dtype=cache_dtype)
    compute.sync()
    got = out.cpu().numpy()
    for b, n in enumerate(lens):
        check(got[b:b + 1], *kinds[n][2], f"sequence {b} of {n}, 2^{bits}")


def small_query_case(rng, n, rows, hq, hkv, d, cache_dtype, magnitude):
    """Queries of the given magnitude (with one element of every head much larger than the others in half of the heads) over keys
    whose scales make up for it."""
    t, blocks = _table(rng, [n], 16)
    (kc, ks), (vc, vs) = (R.random_pool(rng, blocks, 16, hkv, d, cache_dtype) for _ in range(2))
    q = (rng.standard_normal((rows, hq, d)) * magnitude).astype(np.float32)
    q[:, ::2, 3] *= 30
    return t, blocks, q, kc, (ks / np.float32(magnitude)).astype(np.float32), vc, vs


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [0, 1])
@pytest.mark.parametrize("hq,hkv,d,n", [(8, 2, 128, 700), (32, 4, 64, 100), (16, 1, 128, 1500)])
@pytest.mark.parametrize("magnitude", [1e-2, 1e-4, 1e-9, 1e-20, 1e-30, 1e6, 1e30])
def test_decode_q8_queries_of_any_magnitude(compute, cache_dtype, hq, hkv, d, n, magnitude):
    """q . k is the same product whichever of the two holds the magnitude."""
    import torch
    rng = np.random.default_rng(n)
    t, blocks, q, kc, ks, vc, vs = small_query_case(rng, n, 1, hq, hkv, d, cache_dtype, magnitude)
    ref = weighted_reference(q.astype(np.float64), kc, ks, vc, vs, [n - 1], d ** -0.5, cache_dtype, t[0])
    out = torch.full(q.shape, float("nan"), device=DEV)
    compute.batched_paged_attention_decode_q8(*[_dev(x) for x in (q, kc, vc, ks, vs, t)], _dev(np.array([n], np.int32)), out, 1, hq, hkv, d, 16, t.shape[1],
                                              d ** -0.5, num_blocks=blocks, cache_dtype=cache_dtype)
    compute.sync()
    check(out.cpu().numpy(), *ref, f"{magnitude}")


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [0, 1])
@pytest.mark.parametrize("hq,hkv,d,seq,start", [(8, 2, 128, 130, 300), (32, 4, 64, 3, 60), (2, 1, 128, 257, 0)])
@pytest.mark.parametrize("magnitude", [1e-2, 1e-4, 1e-9, 1e-20, 1e-30, 1e6, 1e30])
def test_prefill_q8_queries_of_any_magnitude(compute, cache_dtype, hq, hkv, d, seq, start, magnitude):
    import torch
    rng = np.random.default_rng(seq)
    n = seq + start
    t, blocks, q, kc, ks, vc, vs = small_query_case(rng, n, seq, hq, hkv, d, cache_dtype, magnitude)
    ref = weighted_reference(q.astype(np.float64), kc, ks, vc, vs, start + np.arange(seq), d ** -0.5, cache_dtype, t[0])
    out = torch.full(q.shape, float("nan"), device=DEV)
    compute.paged_prefill_attention_q8(*[_dev(x) for x in (q, kc, vc, ks, vs, t)], out, hq, hkv, seq, start, d, 16, t.shape[1], blocks, d ** -0.5, cache_dtype)
    compute.sync()
    check(out.cpu().numpy(), *ref, f"{magnitude}")


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [0, 1])
def test_prefill_q8_a_query_that_is_not_finite_spoils_its_own_row_and_head(compute, cache_dtype):
    import torch
    rng = np.random.default_rng(8)
    hq, hkv, d, seq, start = 4, 2, 128, 140, 100
    t, blocks, q, kc, ks, vc, vs = small_query_case(rng, seq + start, seq, hq, hkv, d, cache_dtype, 1.0)
    bad = q.copy()
    bad[5, 1, 7], bad[130, 2, 0], bad[131, 0, :] = np.nan, np.inf, 0
    want, bound, norm = weighted_reference(np.where(np.isfinite(bad), bad, 0).astype(np.float64), kc, ks, vc, vs, start + np.arange(seq), d ** -0.5, cache_dtype, t[0])
    out = torch.zeros(q.shape, device=DEV)
    compute.paged_prefill_attention_q8(*[_dev(x) for x in (bad, kc, vc, ks, vs, t)], out, hq, hkv, seq, start, d, 16, t.shape[1], blocks, d ** -0.5, cache_dtype)
    compute.sync()
    got = out.cpu().numpy()
    assert not np.isfinite(got[5, 1]).any() and not np.isfinite(got[130, 2]).any()
    for r, h in ((5, 1), (130, 2)):
        got[r, h] = want[r, h]
    check(got, want, bound, norm, "the other rows and heads")


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", [0, 1])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("k_scale", [0.0, 1e-7, 1e-30, 2.0 ** -126])
def test_prefill_q8_rows_of_zeros_meet_pages_of_zeros(compute, cache_dtype, half, d, k_scale):
    """Query rows of zeros (padding), pages of zero or next to zero keys, in tiles whose later keys are masked: the factor that takes a masked
    score to the base-2 exponent must not vanish.  A row of zeros is the mean of what it sees."""
    import torch
    rng = np.random.default_rng(d)
    hq, hkv, seq, start = 4, 2, 150, 40
    n = seq + start
    t, blocks, q, kc, ks, vc, vs = small_query_case(rng, n, seq, hq, hkv, d, cache_dtype, 1.0)
    kc, ks = kc.copy(), ks.copy()
    q[3], q[64:70, 1], q[149] = 0, 0, 0
    q[80] *= 1e-20 if not half else 0
    if half:
        q = q.astype(np.float16).astype(np.float32)
    for p in (0, 4, 5, 9, 11):
        e = t[0, p]
        ks[e] = k_scale
        if k_scale == 0:
            kc[e * 16:e * 16 + 16] = 0
    ref = weighted_reference(q.astype(np.float64), kc, ks, vc, vs, start + np.arange(seq), d ** -0.5, cache_dtype, t[0])
    dt = torch.float16 if half else torch.float32
    out = torch.full(q.shape, float("nan"), device=DEV)
    compute.paged_prefill_attention_q8(_dev(q, dt), *[_dev(x) for x in (kc, vc, ks, vs, t)], out, hq, hkv, seq, start, d, 16, t.shape[1], blocks, d ** -0.5, cache_dtype,
                                       q_dtype=int(half), out_dtype=0)
    compute.sync()
    check(out.cpu().numpy(), *ref, f"K scale {k_scale}")
