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
