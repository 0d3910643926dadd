"""Plain 64-bit forms of the attention calls that see the cache through a view (8-bit codes with page scales, a
sliding window with sinks), and the bounds that their fp32 results are held to."""
import numpy as np

QMAX = {0: 127.0, 1: 448.0}  # by cache_dtype: int8, fp8 e4m3


def e4m3_values():
    """The 256 codes' values (NaN at 0x7F and 0xFF), from the format: sign, 4 exponent bits (bias 7), 3 mantissa bits."""
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m / 8.0 * 2.0 ** -6, (1 + m / 8.0) * 2.0 ** (e - 7.0))
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b & 128, -v, v)


def decode_codes(codes, cache_dtype):
    """uint8 codes -> float64 values."""
    return codes.view(np.int8).astype(np.float64) if cache_dtype == 0 else e4m3_values()[codes]


def encode(x, cache_dtype):
    """float64 values -> uint8 codes, nearest with ties to even."""
    x = np.asarray(x, np.float64)
    if cache_dtype == 0:
        return np.clip(np.rint(x), -127, 127).astype(np.int8).view(np.uint8)
    table = e4m3_values()[:127]  # 0 .. 448, ascending
    a = np.minimum(np.abs(x), 448.0)
    i = np.clip(np.searchsorted(table, a, side="right") - 1, 0, 125)
    mid = (table[i] + table[i + 1]) / 2
    up = (a > mid) | ((a == mid) & (i % 2 == 1))
    return ((i + up) | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def random_pool(rng, num_blocks, block_size, hkv, d, cache_dtype):
    """Codes over the whole range with page scales that differ by up to 16 times."""
    n = (num_blocks * block_size, hkv, d)
    # (drawn from 4096 encoded values: encoding a whole pool here would be most of a test's time)
    some = encode(np.clip(rng.standard_normal(4096) * 0.3, -1, 1) * QMAX[cache_dtype], cache_dtype)
    codes = some[rng.integers(0, 4096, n, dtype=np.int16)]
    scales = (2.0 ** rng.uniform(-2, 2, (num_blocks, hkv)) * 3.0 / QMAX[cache_dtype]).astype(np.float32)
    return codes, scales


def pool_values(codes, scales, cache_dtype, block_size):
    v = decode_codes(codes, cache_dtype)
    return v * np.repeat(scales.astype(np.float64), block_size, axis=0)[:, :, None]


def rows_of(values, table, n, block_size):
    """Rows 0 .. n-1 of one sequence (entries of pages that are never used may be anything): [n, Hkv, D]."""
    pos = np.arange(n)
    page = np.where(table < 0, 0, table)[pos // block_size]
    return values[page * block_size + pos % block_size]


def visible(pos, n, window, sinks):
    """[len(pos), n] truth: key j may be seen from position pos."""
    p, j = np.asarray(pos)[:, None], np.arange(n)[None, :]
    seen = j <= p
    return seen & ((p - j < window) | (j < sinks)) if window else seen


def attend(q, k, v, pos, scale, window=0, sinks=0):
    """q [R, Hq, D] at positions pos [R] over k, v [n, Hkv, D], all in 64 bits.  Returns the output and, elementwise, the
    bound on what fp32 arithmetic may add: with S the largest sum |q_d k_d| * scale, a score is off by at most
    (D + 8) 2^-24 S (its fp32 sum, and the fp16 hi + lo form of q, which is within 2^-22), a weight by that and 2^-21
    for its exponential and hi + lo form, and the two sums over n weights by n 2^-24 each; relative errors of the weights move a
    weighted mean by at most twice themselves times the largest |v|."""
    import torch
    rows, hq, d = q.shape
    n, hkv = k.shape[:2]
    if n == 0 or rows == 0:
        return np.zeros((rows, hq, d)), np.zeros((rows, hq, 1))
    dev = "cuda" if torch.cuda.is_available() else "cpu"  # elementary float64 products and sums only
    qt = torch.from_numpy(np.ascontiguousarray(q)).to(dev).transpose(0, 1).reshape(hkv, -1, d)         # [Hkv, G * R, D]
    kt, vt = (torch.from_numpy(np.ascontiguousarray(x)).to(dev).transpose(0, 1) for x in (k, v))        # [Hkv, n, D]
    seen = torch.from_numpy(visible(pos, n, window, sinks)).to(dev)
    hidden = ~seen.repeat(hq // hkv, 1)                                                                 # [G * R, n]
    x = torch.matmul(qt, kt.transpose(1, 2)) * scale
    x.masked_fill_(hidden, -float("inf"))
    m = x.amax(-1, keepdim=True)
    w = torch.exp(x - torch.where(torch.isfinite(m), m, 0.0))
    total = w.sum(-1, keepdim=True)
    vt = torch.where(seen.any(0)[None, :, None], vt, 0.0)
    out = torch.matmul(w, vt) / torch.where(total > 0, total, 1.0)
    big = (torch.matmul(qt.abs(), kt.abs().transpose(1, 2)) * scale).masked_fill_(hidden, 0.0).amax(-1, keepdim=True)
    bound = 2 * ((d + 8) * 2.0 ** -24 * big + 2.0 ** -21 + n * 2.0 ** -23) * vt.abs().amax((1, 2), keepdim=True)
    return tuple(t.reshape(hq, rows, -1).transpose(0, 1).cpu().numpy() for t in (out, bound))


def assert_close(got, want, bound, half=False, what=""):
    """Within the elementwise bound (and, for fp16 outputs, half an fp16 step more), and within sqrt(2^15) 2^-24 of the
    result's norm: rounding errors of sums of at most 2^15 terms add up like a random walk."""
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape and np.isfinite(got).all(), what
    limit = np.broadcast_to(bound, want.shape) + (np.abs(want) * 2.0 ** -11 + 2.0 ** -25 if half else 0.0)
    worst = np.abs(got - want) - limit
    assert worst.max(initial=0.0) <= 0, f"{what}: off by {np.abs(got - want).max():.3e}, {worst.max():.3e} over the bound"
    norm = np.linalg.norm(want)
    rel = np.linalg.norm(got - want) / norm if norm else 0.0
    assert rel <= (2.0 ** -11 if half else 2.0 ** -16.5), f"{what}: relative error {rel:.3e}"
