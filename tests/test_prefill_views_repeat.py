"""Prefill with a window or over the 8-bit cache gives the same bits every time, and fp32 results that are off by little more than the sums
in a tensor-core accumulator."""
import numpy as np
import pytest

DEV = "cuda:0"

CASES = [("contiguous", 400, 0, 32, 8, 128, 100, 4), ("contiguous", 2048, 0, 32, 8, 128, 512, 0), ("paged", 1001, 1099, 32, 8, 128, 700, 4), ("paged", 300, 900, 8, 2, 64, 100, 20),
         ("int8", 509, 1531, 32, 8, 128, 0, 0), ("e4m3", 200, 4000, 8, 2, 64, 0, 0), ("int8", 700, 6000, 16, 4, 128, 3000, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,seq,start,hq,hkv,d,window,sinks", CASES)
@pytest.mark.parametrize("half", [False, True])
def test_prefill_repeats_bit_for_bit_and_close(compute, kind, seq, start, hq, hkv, d, window, sinks, half):
    import torch
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seq)
    n = seq + start
    blocks = (n + 15) // 16
    dt = torch.float16 if half else torch.float32
    q = torch.empty((seq, hq, d), device=DEV).normal_(generator=gen).to(dt)
    table = torch.randperm(blocks, device=DEV, generator=gen).int()
    rows = (table.long()[:, None] * 16 + torch.arange(16, device=DEV)).flatten()[:n]
    common = dict(q_dtype=int(half), out_dtype=int(half))

    def normal(*shape):
        return torch.empty(shape, device=DEV).normal_(generator=gen)

    if kind == "contiguous":
        k, v = normal(hkv, n, d).half(), normal(hkv, n, d).half()
        kd, vd = k.double(), v.double()
        run = lambda out: compute.multihead_attention_window(q, k, v, out, hq, hkv, seq, n, d, d ** -0.5, window, sinks, start_pos=start, **common)
    elif kind == "paged":
        k, v = normal(blocks * 16, hkv, d).half(), normal(blocks * 16, hkv, d).half()
        kd, vd = (x[rows].double().transpose(0, 1) for x in (k, v))
        run = lambda out: compute.paged_prefill_attention_window(q, k, v, table, out, hq, hkv, seq, start, d, 16, blocks, blocks, d ** -0.5, window, sinks, **common)
    else:
        code = torch.int8 if kind == "int8" else torch.float8_e4m3fn
        k, v = ((normal(blocks * 16, hkv, d) * (32 if kind == "int8" else 112)).clamp(-127, 127).to(code) for _ in range(2))
        ks, vs = (((0.5 + torch.rand((blocks, hkv), device=DEV, generator=gen)) / 32) for _ in range(2))
        kd, vd = ((x.float().double() * s.double().repeat_interleave(16, 0)[:, :, None])[rows].transpose(0, 1) for x, s in ((k, ks), (v, vs)))
        run = lambda out: compute.paged_prefill_attention_q8(q, k, v, ks, vs, table, out, hq, hkv, seq, start, d, 16, blocks, blocks, d ** -0.5, int(kind == "e4m3"),
                                                             window=window, sinks=sinks, **common)
    outs = [torch.full((seq, hq, d), float("nan"), device=DEV, dtype=dt) for _ in range(12)]
    for out in outs:
        run(out)
    compute.sync()
    assert all(torch.equal(outs[0], o) for o in outs[1:])
    pos, j = start + torch.arange(seq, device=DEV)[:, None], torch.arange(n, device=DEV)
    seen = (j <= pos) & ((pos - j < window) | (j < sinks)) if window else j <= pos
    want = torch.empty((seq, hq, d), device=DEV, dtype=torch.float64)
    for h in range(hq):
        x = (q[:, h].double() @ kd[h // (hq // hkv)].T) * d ** -0.5
        want[:, h] = torch.softmax(x.masked_fill_(~seen, -float("inf")), -1) @ vd[h // (hq // hkv)]
    rel = float((outs[0].double() - want).norm() / want.norm())
    # A truncated addition is off by half a unit in the last place of the sum on average, 2^-24 of it, and all one way: over the eight additions of a
    # tile, and a sum that grows evenly (half its end on average), 2^-22 of the result per tile; 22 tiles at most, and 2^-20 for all else
    # (scores, weights and their fp16 hi + lo form, the merge).  fp16 outputs: half a step more.
    assert rel <= 22 * 2.0 ** -22 + 2.0 ** -20 + (2.0 ** -11 if half else 0.0), rel
    if not half:
        assert rel <= min(22, (n + 127) // 128) * 2.0 ** -22 + 2.0 ** -20, rel
