"""The index arithmetic behind the windowed and 8-bit calls (csrc/view_plan.h, the header that the kernels are compiled from), run on
the host against the definitions.  Built with the sanitizer for undefined arithmetic: an overflow ends the test."""
import ctypes as C
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

import view_reference as R

SOURCE = Path(__file__).resolve().parent / "host_drivers" / "view_plan.cpp"


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    lib = tmp_path_factory.mktemp("view_plan") / "view_plan.so"
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-fsanitize=signed-integer-overflow", "-fsanitize-undefined-trap-on-error", "-shared", "-fPIC",
                    "-o", str(lib), str(SOURCE)], check=True)
    return C.CDLL(str(lib))


def _ints(fn, n, *args):
    out = (C.c_int * n)()
    fn(*args, out)
    return list(out)


def test_window_span_is_the_definition(plans):
    for window in (0, 1, 2, 5, 16, 100, 0x7fffffff):
        for sinks in (0, 1, 7, 40, 0x7fffffff):
            for pos in range(0, 60):
                end, lo = _ints(plans.view_window_span, 2, pos, window, sinks)
                assert 0 <= end <= lo or lo == end == 0
                keys = sorted(set(range(end)) | set(range(lo, pos + 1)))
                assert np.array_equal(np.nonzero(R.visible([pos], pos + 1, window, sinks)[0])[0], keys)
    assert _ints(plans.view_window_span, 2, 2 ** 31 - 65537, 7, 0x7fffffff) == [2 ** 31 - 65543] * 2


def test_window_steps_walk_every_visible_tile_once(plans):
    rng = np.random.default_rng(1)
    for i in range(400):
        seq_q, start = int(rng.integers(1, 700)), int(rng.choice([0, rng.integers(0, 2000)]))
        end = start + seq_q
        seq_kv = end if i % 3 else max(1, end - int(rng.integers(0, 900)))
        window = int(rng.choice([0, 1, 17, 128, rng.integers(1, 1500), 0x7fffffff]))
        sinks = int(rng.choice([0, 3, 128, 200, rng.integers(0, 900), 0x7fffffff])) if window else 0
        for q0 in range(0, seq_q, 128):
            pos = start + np.arange(q0, min(q0 + 128, seq_q))
            seen = R.visible(pos, seq_kv, window, sinks).any(0)
            n, n_sink, w0, lo = _ints(plans.view_window_steps, 4, seq_q, seq_kv, start, window, sinks, q0)
            tiles = [j if j < n_sink else j - n_sink + w0 for j in range(n)]
            assert n >= 1 and tiles == sorted(set(tiles))
            need = sorted(set(np.nonzero(seen)[0] // 128))
            # every tile with a visible key, and no other: but for the tile that a cache ends in before the window begins, and for the one
            # step of a block that sees nothing
            assert set(need) <= set(tiles) and set(tiles) - set(need) <= ({seq_kv // 128} if need and lo >= seq_kv else set() if need else {0, seq_kv // 128})
            hidden = np.nonzero(~seen[: min(lo, seq_kv)])[0]
            assert np.array_equal(hidden, np.arange(min(sinks, lo, seq_kv), min(lo, seq_kv)))  # what the kernel clears


def test_chunks_share_out_every_step(plans):
    for n in (1, 2, 5, 31, 32, 33, 1000, 1 << 24):
        for chunks in (1, 2, 3, 24, 32):
            at = [plans.view_chunk_begin(n, chunks, c) for c in range(chunks + 1)]
            assert at[0] == 0 and at[-1] == n and all(0 <= b - a <= -(-n // chunks) for a, b in zip(at, at[1:]))


def test_append_rows_cover_what_can_be_placed_and_nothing_else(plans):
    """Every start a 32-bit position can name, the ends of the range among them: the pages that a call touches (as many as the launch has
    blocks for) hold exactly the positions of [start, start + new_len) that lie in [0, room)."""
    fn = plans.view_append_rows
    rng = np.random.default_rng(2)
    far = [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 200, 2 ** 30, -1, -7, -300, -(2 ** 31)]
    for bs in (1, 5, 16, 48, 1 << 20):
        for new_len in (1, 2, 16, 17, 300):
            for start in far + [0, 1, 15, 16, 47, 63, 64] + [int(x) for x in rng.integers(0, 400, 5)]:
                room = int(rng.integers(1, 400))
                pages = (new_len + bs - 2) // bs + 1
                got = []
                for i in range(pages):
                    out = (C.c_longlong * 3)()
                    fn(C.c_longlong(start), C.c_longlong(new_len), C.c_longlong(room), bs, i, out)
                    page, r0, r1 = out
                    assert 0 <= r0 <= bs and 0 <= r1 <= bs
                    if r0 < r1:
                        assert 0 <= page <= (room - 1) // bs
                        got += range(page * bs + r0, page * bs + r1)
                assert got == list(range(max(start, 0), max(min(start + new_len, room), max(start, 0))))


def _plan(plans, seq_q, start, heads, head_dim=128, out_fp16=False, window=0, sinks=0, batch=1, seq_kv=None, sms=148):
    shape = (C.c_int * 10)(seq_q, seq_kv or start + seq_q, start, window, sinks, batch, heads, head_dim, sms, int(out_fp16))
    out = (C.c_longlong * 5)()
    plans.view_chunk_plan(shape, out)
    return dict(zip(("wanted", "rows", "longest", "chunks", "bytes"), out))


LONG = [(16384, 114688, 64), (32768, 98304, 32), (8192, 57344, 64), (2048, 129024, 32), (2048, 14336, 32), (4001, 4099, 32), (509, 1531, 32), (1, 1000000, 8),
        (131072, 0, 128), (128, 2000000, 65535), (100, 0, 4)]


@pytest.mark.parametrize("seq_q,start,heads", LONG)
@pytest.mark.parametrize("out_fp16", [False, True])
@pytest.mark.parametrize("window,sinks", [(0, 0), (4096, 4), (100000, 1000)])
def test_chunk_plans_bound_the_run_of_an_accumulator_and_the_partials(plans, seq_q, start, heads, out_fp16, window, sinks):
    """No launch holds more than a GiB of partials; an accumulator takes 22 key tiles for an fp32 output and 128 for an fp16 one, or - over more
    tiles than 32 chunks of those - a 32nd of the tiles; only where 128 rows of partials pass the limit by themselves are there fewer chunks,
    and then the most that fit."""
    p = _plan(plans, seq_q, start, heads, out_fp16=out_fp16, window=window, sinks=sinks)
    tiles = 128 if out_fp16 else 22
    assert p["bytes"] <= 1 << 30
    assert p["rows"] == seq_q or p["rows"] % 128 == 0 and 0 < p["rows"] < seq_q
    steps = -(-p["longest"] // p["chunks"])
    row_bytes = heads * (128 * 4 + 8) * 128
    if row_bytes * p["wanted"] <= 1 << 30:
        assert steps <= max(tiles, -(-p["longest"] // 32)), (p, steps)
    else:
        fits = [n for n in (1, 2, 3, 4, 6, 8, 12, 16, 24, 32) if n == 1 or row_bytes * n <= 1 << 30]
        assert p["rows"] == min(128, seq_q) and p["chunks"] == max(fits)
    # rows are only given to several launches when they have to be
    if p["rows"] < seq_q:
        assert heads * (128 * 4 + 8) * seq_q * p["wanted"] > 1 << 30
        assert p["rows"] == 128 or heads * (128 * 4 + 8) * (p["rows"] + 128) * p["wanted"] > 1 << 30


def test_chunk_plans_of_short_calls_stay_in_one_launch(plans):
    for seq_q, start, heads, window in ((2048, 0, 32, 512), (509, 1531, 32, 0), (4001, 4099, 32, 2047), (2048, 14336, 32, 0)):
        assert _plan(plans, seq_q, start, heads, window=window)["rows"] == seq_q
