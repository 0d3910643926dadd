"""The compute object's workspaces: what happens to them when they grow, around captured graphs and near the end of the memory."""
import numpy as np
import pytest

import view_reference as R
from granite_b200 import synth
from test_q8_cache import _decode_case, _dev

DEV = "cuda:0"


def _q8_step(o, held, c, out, hq, hkv, d):
    o.batched_paged_attention_decode_q8(*held, out, len(c["lens"]), hq, hkv, d, 16, c["tables"].shape[1], c["scale"], num_blocks=c["blocks"], cache_dtype=0)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["relaxed", "thread_local"])
@pytest.mark.parametrize("warm", ["nothing", "scratch"])
def test_workspaces_do_not_grow_inside_a_capture(mode, warm):
    """A relaxed capture allows allocations, but clearing the page counters would become a node of the graph, and calls before its first
    replay would count in whatever the new memory holds.  The call is refused, the capture goes on, and the object works."""
    import torch
    import granite_b200 as g
    hq, hkv, d = 32, 8, 128
    side = torch.cuda.Stream(device=DEV)
    o = g.CudaCompute(0, side.cuda_stream)
    c = _decode_case(80, [900, 1200, 40] * 20, hq, hkv, d, 0)  # 60 sequences: planned and merged inside the decode kernel
    held = [_dev(c[n]) for n in ("q", "kc", "vc", "ks", "vs", "tables", "lens")]
    out, mark = torch.zeros(c["q"].shape, device=DEV), torch.zeros(8, device=DEV)
    plain = synth.paged_case(81, 60, 200, 1500, hq, hkv, d, device=DEV)
    p_tables, p_lens = torch.from_numpy(plain.tables).to(DEV), torch.from_numpy(plain.seq_lens).to(DEV)
    p_out = [torch.zeros((60, hq, d), device=DEV) for _ in range(2)]

    def plain_step(obj, where):
        obj.batched_paged_attention_decode(plain.q, plain.k_pool, plain.v_pool, p_tables, p_lens, where, 60, hq, hkv, d, synth.PAGE, plain.max_blocks, d ** -0.5,
                                           num_blocks=plain.num_blocks)

    if warm == "scratch":  # enough scratch for the step, but no page counters yet
        q = torch.zeros((1024, hq, d), device=DEV)
        kv = torch.zeros((hkv, 1024, d), device=DEV).half()
        o.multihead_attention(q, kv, kv, torch.empty_like(q), hq, hkv, 1024, 1024, d, d ** -0.5, 1024)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side, capture_error_mode=mode):
        mark.add_(1)
        for call in (lambda: _q8_step(o, held, c, out, hq, hkv, d), lambda: plain_step(o, p_out[0])):
            with pytest.raises(g.GraniteCudaError) as e:
                call()
            assert e.value.code == g.ErrorCode.InvalidState and "captur" in str(e.value)
    # eager calls before any replay, on counters that a junk-filled pool could have given
    _q8_step(o, held, c, out, hq, hkv, d)
    plain_step(o, p_out[0])
    o.sync()
    R.assert_close(out.cpu().numpy(), c["want"], c["bound"], what="eager after the capture")
    fresh = g.CudaCompute(0)
    torch.cuda.synchronize()
    plain_step(fresh, p_out[1])
    fresh.sync()
    assert torch.equal(p_out[0], p_out[1])
    graph.replay()
    torch.cuda.synchronize()
    assert mark.cpu().tolist() == [1.0] * 8
    # warm now: the same call can be captured
    out.zero_()
    torch.cuda.synchronize()
    graph2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph2, stream=side, capture_error_mode=mode):
        _q8_step(o, held, c, out, hq, hkv, d)
    graph2.replay()
    torch.cuda.synchronize()
    R.assert_close(out.cpu().numpy(), c["want"], c["bound"], what="replay")
    del graph, graph2
    o.shutdown()
    fresh.shutdown()


@pytest.mark.gpu
def test_scratch_grows_in_place_near_the_end_of_the_memory():
    """Growing needs room for the new arena, not for both.  What room is left is what the first arena and the calls need, less than the
    second arena takes by itself."""
    import torch
    import granite_b200 as g
    torch.cuda.empty_cache()
    hq, hkv, d = 32, 8, 128
    o = g.CudaCompute(0)
    kv = torch.randn((hkv, 256, d), device=DEV).half()
    rows = (16384, 24576, 65536)  # 335, 503 and 1342 MB of scratch: fp16 hi + lo, and a quarter more
    q = torch.randn((rows[2], hq, d), device=DEV)
    out = torch.zeros_like(q)

    def call(n):  # prompt rows far behind a short cache: every row sees all 256 keys
        o.multihead_attention(q, kv, kv, out, hq, hkv, n, 256, d, d ** -0.5, 256, start_pos=256)
        o.sync()

    torch.cuda.synchronize()
    call(rows[0])
    want = out[:rows[0]].cpu()
    room = 400 << 20
    hog = torch.empty(torch.cuda.mem_get_info(0)[0] - room, dtype=torch.uint8, device=DEV)
    try:
        assert torch.cuda.mem_get_info(0)[0] < rows[1] * hq * d * 5
        out.zero_()
        torch.cuda.synchronize()
        call(rows[1])
        assert torch.allclose(out[:rows[0]].cpu(), want, rtol=1e-4, atol=1e-6)
        # no room at all: refused, and the object works once there is
        with pytest.raises(g.GraniteCudaError) as e:
            call(rows[2])
        assert e.value.code == g.ErrorCode.OutOfMemory
        call(rows[0])
    finally:
        del hog
        torch.cuda.empty_cache()
    call(rows[2])
    assert torch.allclose(out[:rows[0]].cpu(), want, rtol=1e-4, atol=1e-6) and bool(torch.isfinite(out).all())
    o.shutdown()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["contiguous", "paged", "q8"])
def test_a_prefill_of_many_rows_over_a_long_context_runs_in_several_launches(kind):
    """4096 fp32 rows of 64 heads over 100000 keys want 32 chunks each: more partials than a launch may hold.  The scratch stays bounded, and the
    rows on both sides of the cuts come out right."""
    import torch
    import granite_b200 as g
    hq, hkv, d, seq, start = 64, 1, 64, 4096, 96000
    n, scale, window, sinks = seq + start, d ** -0.5, 99000, 8
    gen = torch.Generator(device=DEV)
    gen.manual_seed(3)
    q = torch.empty((seq, hq, d), device=DEV).normal_(generator=gen)
    kv = [torch.empty((1, n, d), device=DEV).normal_(generator=gen).half() for _ in range(2)]
    out = torch.full_like(q, float("nan"))
    blocks = (n + 15) // 16
    table = torch.randperm(blocks, device=DEV, generator=gen).int()
    o = g.CudaCompute(0)
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info(0)[0]
    if kind == "contiguous":
        o.multihead_attention_window(q, *kv, out, hq, hkv, seq, n, d, scale, window, sinks, start_pos=start)
    elif kind == "paged":
        pools = []
        for x in kv:
            p = torch.zeros((blocks, 16, 1, d), device=DEV, dtype=torch.float16)
            p[table.long()] = torch.nn.functional.pad(x[0], (0, 0, 0, blocks * 16 - n)).view(blocks, 16, 1, d)
            pools.append(p)
        torch.cuda.synchronize()
        free = torch.cuda.mem_get_info(0)[0]
        o.paged_prefill_attention_window(q, *pools, table, out, hq, hkv, seq, start, d, 16, blocks, blocks, scale, window, sinks)
    else:
        codes = [(x[0].float() * 30).round().clamp(-127, 127).to(torch.int8) for x in kv]
        kv = [(c.double() / 30)[None] for c in codes]
        pools = []
        for c in codes:
            p = torch.zeros((blocks, 16, 1, d), device=DEV, dtype=torch.int8)
            p[table.long()] = torch.nn.functional.pad(c, (0, 0, 0, blocks * 16 - n)).view(blocks, 16, 1, d)
            pools.append(p)
        scales = torch.full((blocks, 1), 1 / 30, device=DEV)
        torch.cuda.synchronize()
        free = torch.cuda.mem_get_info(0)[0]
        o.paged_prefill_attention_q8(q, *pools, scales, scales, table, out, hq, hkv, seq, start, d, 16, blocks, blocks, scale, 0, window=window, sinks=sinks)
    o.sync()
    # partials of 1 GiB, the queries' halves, the 8-bit cache's fp16 copy, a quarter more
    assert free - torch.cuda.mem_get_info(0)[0] <= 1.25 * ((1 << 30) + q.numel() * 4 + 4 * n * d + (1 << 20)) + (64 << 20)
    k, v = (x[0].double() for x in kv)
    for rows in (slice(0, 3), slice(seq - 2 * 1920 - 5, seq - 2 * 1920 + 5), slice(seq - 1925, seq - 1915), slice(seq - 3, seq)):
        pos = start + torch.arange(seq, device=DEV)[rows]
        j = torch.arange(n, device=DEV)
        seen = (j <= pos[:, None]) & ((pos[:, None] - j < window) | (j < sinks))
        x = torch.einsum("rhd,nd->rhn", q[rows].double(), k) * scale
        x.masked_fill_(~seen[:, None], -float("inf"))
        w = torch.softmax(x, -1)
        want, mean = w @ v, w @ v.abs()
        # a 32nd of the tiles in one accumulator, 2.4e-9 for each key, and what any of the calls may be off by (view_reference.assert_close)
        assert ((out[rows].double() - want).abs() <= mean * (2.4e-9 * n / 32 + 2.0 ** -16.5)).all()
    o.shutdown()


@pytest.mark.gpu
def test_a_prefill_without_room_for_partials_runs_in_one_chunk():
    """Few rows over a long context are cut along the keys where the scratch has room, and run in one piece where it has not."""
    import torch
    import granite_b200 as g
    torch.cuda.empty_cache()
    hq, hkv, d, seq, n = 32, 8, 128, 2048, 16384
    q = torch.randn((seq, hq, d), device=DEV).half()
    k, v = (torch.randn((hkv, n, d), device=DEV).half() for _ in range(2))
    outs = [torch.zeros((seq, hq, d), device=DEV) for _ in range(2)]

    def call(o, out):
        o.multihead_attention_window(q, k, v, out, hq, hkv, seq, n, d, d ** -0.5, n, 0, q_dtype=1, start_pos=n - seq)
        o.sync()

    roomy, tight = g.CudaCompute(0), g.CudaCompute(0)
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info(0)[0]
    call(roomy, outs[0])
    assert before - torch.cuda.mem_get_info(0)[0] > 150 << 20  # at least six chunks of 34 MB
    hog = torch.empty(torch.cuda.mem_get_info(0)[0] - (120 << 20), dtype=torch.uint8, device=DEV)
    try:
        call(tight, outs[1])
    finally:
        del hog
        torch.cuda.empty_cache()
    # one run over 128 tiles: 2.4e-9 a key
    assert float((outs[0] - outs[1]).norm() / outs[0].norm()) <= 2.4e-9 * n
    roomy.shutdown()
    tight.shutdown()


@pytest.mark.gpu
def test_a_prefill_of_several_launches_is_captured_whole_or_not_at_all():
    """Every launch of it needs scratch of its own size, the one over the last rows the most: where the arena cannot grow, nothing is captured of
    the call."""
    import torch
    import granite_b200 as g
    hq, hkv, d, seq, start = 64, 1, 64, 2500, 96000
    n = seq + start
    blocks = (n + 15) // 16
    side = torch.cuda.Stream(device=DEV)
    o = g.CudaCompute(0, side.cuda_stream)
    gen = torch.Generator(device=DEV)
    gen.manual_seed(5)
    q = torch.empty((seq, hq, d), device=DEV).normal_(generator=gen)
    k, v = (torch.randint(-127, 128, (blocks * 16, hkv, d), device=DEV, generator=gen, dtype=torch.int8) for _ in range(2))
    scales = torch.full((blocks, hkv), 1 / 40, device=DEV)
    table = torch.arange(blocks, device=DEV, dtype=torch.int32)
    outs = [torch.zeros_like(q) for _ in range(2)]

    def call(out, rows, first):
        o.paged_prefill_attention_q8(q[first:first + rows], k, v, scales, scales, table, out[first:first + rows], hq, hkv, rows, start + first, d, 16, blocks, blocks,
                                     d ** -0.5, 0)

    torch.cuda.synchronize()
    call(outs[0], 1000, 0)  # half of what the call's launches need
    o.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side, capture_error_mode="relaxed"):
        before = o.get_profiling_stats()[0]
        with pytest.raises(g.GraniteCudaError) as e:
            call(outs[1], seq, 0)
        assert e.value.code == g.ErrorCode.InvalidState and o.get_profiling_stats()[0] == before
    call(outs[1], seq, 0)  # two launches, over rows 580 to 2499 and 0 to 579
    o.sync()
    outs[1].zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side, capture_error_mode="relaxed"):
        call(outs[1], seq, 0)
    graph.replay()
    torch.cuda.synchronize()
    call(outs[0], 1500, 1000)
    o.sync()
    # (the two are cut elsewhere along the rows and keys: equal to the error of their sums)
    assert float((outs[0] - outs[1]).norm() / outs[0].norm()) < 1e-5
    del graph
    o.shutdown()


@pytest.mark.gpu
def test_a_batch_of_long_prefills_runs_sequence_by_sequence():
    """The partials of the batch pass the limit, those of one sequence do not: the same rows as three calls give, in fp32 from fp16 queries."""
    import torch
    import granite_b200 as g
    hq, hkv, d, seq, n, batch = 64, 1, 64, 1500, 98000, 3
    gen = torch.Generator(device=DEV)
    gen.manual_seed(4)
    q = torch.empty((batch, seq, hq, d), device=DEV).normal_(generator=gen).half()
    k, v = (torch.empty((batch, hkv, n, d), device=DEV).normal_(generator=gen).half() for _ in range(2))
    outs = [torch.zeros((batch, seq, hq, d), device=DEV) for _ in range(2)]
    o = g.CudaCompute(0)
    torch.cuda.synchronize()
    args = (hq, hkv, seq, n - 100, d, d ** -0.5, 97000, 4, n)
    before = o.get_profiling_stats()[0]
    o.multihead_attention_window(q, k, v, outs[0], *args, q_dtype=1, start_pos=n - 100 - seq, batch_size=batch)
    assert o.get_profiling_stats()[0] - before == 2 * batch  # attention and merge of each
    for b in range(batch):
        o.multihead_attention_window(q[b], k[b], v[b], outs[1][b], *args, q_dtype=1, start_pos=n - 100 - seq)
    o.sync()
    assert torch.equal(outs[0], outs[1]) and bool(outs[0].any())
    o.shutdown()
