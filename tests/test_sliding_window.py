"""Sliding window with sinks over the fp16 caches: decode and causal prefill, contiguous and paged, against a plain 64-bit
form.  Pages and rows that no query sees are poisoned and their table entries made invalid."""
import ctypes as C

import numpy as np
import pytest

import view_reference as R
from test_q8_cache import _dev, _refusal, _table

DEV = "cuda:0"
WINDOWS = [(1, 0), (1, 1), (16, 0), (17, 5), (64, 16), (100, 33), (100, 200), (127, 129), (128, 128), (300, 4), (0x7fffffff, 0xffffffff)]


def _cache(rng, *shape):
    k, v = (rng.standard_normal(shape, dtype=np.float32).astype(np.float16) for _ in range(2))
    return k, v


def _decode_case(seed, lens, hq, hkv, d, window, sinks):
    rng = np.random.default_rng(seed)
    lens = np.asarray(lens, np.int32)
    tables, blocks = _table(rng, lens, 16)
    k, v = _cache(rng, blocks * 16, hkv, d)
    q = rng.standard_normal((len(lens), hq, d), dtype=np.float32)
    want, bound = np.zeros(q.shape), np.zeros((len(lens), hq, 1))
    live = np.zeros(blocks * 16, bool)
    for b, n in enumerate(lens):
        o, e = R.attend(q[b:b + 1].astype(np.float64), R.rows_of(k, tables[b], n, 16).astype(np.float64),
                        R.rows_of(v, tables[b], n, 16).astype(np.float64), [n - 1], d ** -0.5, window, sinks)
        want[b], bound[b] = o[0], e[0]
        seen = R.visible([n - 1], n, window, sinks)[0] if n else np.zeros(0, bool)
        for j in np.nonzero(seen)[0]:
            live[tables[b, j // 16] * 16 + j % 16] = True
        for pg in range((n + 15) // 16):
            if not seen[pg * 16:pg * 16 + 16].any():
                tables[b, pg] = blocks + 1
    k[~live], v[~live] = np.nan, np.inf
    return q, k, v, tables, lens, blocks, want, bound


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (8, 2, 64), (16, 1, 128), (6, 3, 128), (12, 12, 64), (4, 2, 40)])
@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_paged_decode_window(compute, hq, hkv, d, window, sinks):
    import torch
    q, k, v, tables, lens, blocks, want, bound = _decode_case(d + window % 999, [0, 1, 15, 16, 17, 40, 116, 117, 118, 133, 300, 777], hq, hkv, d, window, sinks)
    out = torch.full(q.shape, float("nan"), device=DEV)
    compute.batched_paged_attention_decode_window(_dev(q), _dev(k), _dev(v), _dev(tables), _dev(lens), out, len(lens), hq, hkv, d, 16, tables.shape[1],
                                                  d ** -0.5, window, sinks, num_blocks=blocks)
    compute.sync()
    got = out.cpu().numpy()
    R.assert_close(got, want, bound, what=f"{window}+{sinks}")
    assert not got[0].any()


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d,lens,window,sinks", [
    (32, 8, 128, [5000], 1024, 4), (32, 8, 128, [8000, 100, 3000], 4000, 40), (16, 2, 128, [5000] * 40, 700, 16), (64, 8, 128, [900, 2000] * 110, 333, 1),
    (8, 8, 64, [3000, 1] * 60, 1000, 0)])
def test_paged_decode_window_batches(compute, hq, hkv, d, lens, window, sinks):
    """One sequence and many: the ways the work is cut."""
    import torch
    q, k, v, tables, lens, blocks, want, bound = _decode_case(len(lens), lens, hq, hkv, d, window, sinks)
    out = torch.full(q.shape, float("nan"), device=DEV)
    for _ in range(2):
        compute.batched_paged_attention_decode_window(_dev(q), _dev(k), _dev(v), _dev(tables), _dev(lens), out, len(lens), hq, hkv, d, 16,
                                                      tables.shape[1], d ** -0.5, window, sinks, num_blocks=blocks)
    compute.sync()
    R.assert_close(out.cpu().numpy(), want, bound, what=f"{window}+{sinks}")


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d,n,max_seq,batch", [(32, 8, 128, 777, 800, 1), (8, 2, 64, 130, 130, 3), (32, 8, 128, 6000, 6001, 1), (4, 4, 128, 1, 5, 2), (4, 2, 40, 99, 100, 2),
                                                      (16, 4, 128, 600, 640, 50)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (33, 3), (128, 0), (500, 70)])
def test_contiguous_decode_window(compute, hq, hkv, d, n, max_seq, batch, window, sinks):
    import torch
    rng = np.random.default_rng(n + window)
    k, v = _cache(rng, batch, hkv, max_seq, d)
    q = rng.standard_normal((batch, hq, d), dtype=np.float32)
    want, bound = np.zeros(q.shape), np.zeros((batch, hq, 1))
    for b in range(batch):
        o, e = R.attend(q[b:b + 1].astype(np.float64), k[b, :, :n].transpose(1, 0, 2).astype(np.float64), v[b, :, :n].transpose(1, 0, 2).astype(np.float64),
                        [n - 1], d ** -0.5, window, sinks)
        want[b], bound[b] = o[0], e[0]
    hidden = ~np.pad(R.visible([n - 1], n, window, sinks)[0], (0, max_seq - n))
    k[:, :, hidden], v[:, :, hidden] = np.nan, np.inf
    out = torch.full(q.shape, float("nan"), device=DEV)
    compute.multihead_attention_window(_dev(q), _dev(k), _dev(v), out, hq, hkv, 1, n, d, d ** -0.5, window, sinks, max_seq, batch_size=batch)
    compute.sync()
    R.assert_close(out.cpu().numpy(), want, bound, what=f"{window}+{sinks}")


PREFILLS = [(2, 0, 8, 2, 128), (127, 1, 4, 1, 128), (128, 0, 8, 2, 64), (129, 127, 8, 2, 128), (300, 333, 6, 3, 128), (400, 0, 4, 4, 64), (65, 700, 32, 8, 128), (20, 50, 4, 2, 40)]


@pytest.mark.gpu
@pytest.mark.parametrize("seq,start,hq,hkv,d", PREFILLS)
@pytest.mark.parametrize("window,sinks,half", [(w, s, bool(i % 2)) for i, (w, s) in enumerate(WINDOWS)])
def test_paged_prefill_window(compute, seq, start, hq, hkv, d, window, sinks, half):
    import torch
    rng = np.random.default_rng(seq + window % 99)
    n = start + seq
    tables, blocks = _table(rng, [n], 16)
    k, v = _cache(rng, blocks * 16, hkv, d)
    dt = np.float16 if half else np.float32
    q = rng.standard_normal((seq, hq, d), dtype=np.float32).astype(dt)
    pos = start + np.arange(seq)
    want, bound = R.attend(q.astype(np.float64), R.rows_of(k.astype(np.float64), tables[0], n, 16), R.rows_of(v.astype(np.float64), tables[0], n, 16), pos,
                           d ** -0.5, window, sinks)
    seen = R.visible(pos, n, window, sinks).any(0)
    live = np.zeros(blocks * 16, bool)
    for j in np.nonzero(seen)[0]:
        live[tables[0, j // 16] * 16 + j % 16] = True
    for pg in range(tables.shape[1]):
        if not seen[pg * 16:pg * 16 + 16].any():
            tables[0, pg] = -5
    k[~live], v[~live] = np.nan, np.inf
    out = torch.full(q.shape, float("nan"), device=DEV, dtype=torch.float16 if half else torch.float32)
    compute.paged_prefill_attention_window(_dev(q), _dev(k), _dev(v), _dev(tables), out, hq, hkv, seq, start, d, 16, tables.shape[1], blocks, d ** -0.5, window,
                                           sinks, q_dtype=int(half), out_dtype=int(half))
    compute.sync()
    R.assert_close(out.float().cpu().numpy(), want, bound, half, f"{seq}@{start} {window}+{sinks}")


@pytest.mark.gpu
@pytest.mark.parametrize("seq,start,hq,hkv,d", PREFILLS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (17, 5), (128, 128), (300, 4)])
@pytest.mark.parametrize("half,batch,short", [(False, 1, 0), (True, 2, 0), (False, 2, 60)])
def test_contiguous_prefill_window(compute, seq, start, hq, hkv, d, window, sinks, half, batch, short):
    """`short`: the cache ends before the last queries' positions, so that some rows may see nothing: they are zero."""
    import torch
    rng = np.random.default_rng(seq + window)
    n = max(start + seq - short, 1)
    max_seq = n + 9
    k, v = _cache(rng, batch, hkv, max_seq, d)
    dt = np.float16 if half else np.float32
    q = rng.standard_normal((batch, seq, hq, d), dtype=np.float32).astype(dt)
    pos = start + np.arange(seq)
    want, bound = np.zeros(q.shape), np.zeros((batch, seq, hq, 1))
    for b in range(batch):
        want[b], bound[b] = R.attend(q[b].astype(np.float64), k[b, :, :n].transpose(1, 0, 2).astype(np.float64), v[b, :, :n].transpose(1, 0, 2).astype(np.float64),
                                     pos, d ** -0.5, window, sinks)
    hidden = ~np.pad(R.visible(pos, n, window, sinks).any(0), (0, max_seq - n))
    k[:, :, hidden], v[:, :, hidden] = np.nan, np.inf
    out = torch.full(q.shape, float("nan"), device=DEV, dtype=torch.float16 if half else torch.float32)
    compute.multihead_attention_window(_dev(q), _dev(k), _dev(v), out, hq, hkv, seq, n, d, d ** -0.5, window, sinks, max_seq, q_dtype=int(half),
                                       out_dtype=int(half), start_pos=start, batch_size=batch)
    compute.sync()
    R.assert_close(out.float().cpu().numpy(), want, bound, half, f"{seq}@{start} {window}+{sinks}")


@pytest.mark.gpu
def test_a_window_that_hides_nothing_is_the_plain_call(compute):
    import torch
    q, k, v, tables, lens, blocks, want, bound = _decode_case(4, [50, 900, 3, 2100], 32, 8, 128, 1 << 20, 3)
    k, v = np.nan_to_num(k), np.where(np.isfinite(v), v, 0)
    outs = [torch.empty(q.shape, device=DEV) for _ in range(2)]
    held = [_dev(x) for x in (q, k, v, tables, lens)]
    compute.batched_paged_attention_decode(*held, outs[0], 4, 32, 8, 128, 16, tables.shape[1], 128 ** -0.5, num_blocks=blocks)
    compute.batched_paged_attention_decode_window(*held, outs[1], 4, 32, 8, 128, 16, tables.shape[1], 128 ** -0.5, 1 << 20, 3, num_blocks=blocks)
    compute.sync()
    for o in outs:
        R.assert_close(o.cpu().numpy(), want, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d", [(16, 4, 128), (8, 2, 128), (4, 1, 128), (16, 4, 64), (8, 2, 64), (4, 1, 64), (24, 2, 64)])
def test_split_pages_of_the_fp16_cache(compute, hq, hkv, d):
    """The plain call and the windowed one where warps share a head's pages: ragged lengths that start segments at odd places of
    the ring and wrap it many times; every run gives the same bits."""
    import torch
    lens = [3001, 17, 2000, 1, 999, 16, 48, 2500, 33] * 6
    for window, sinks in ((0, 0), (1000, 20)):
        q, k, v, tables, ln, blocks, want, bound = _decode_case(hkv + d, lens, hq, hkv, d, window, sinks)
        held = [_dev(x) for x in (q, k, v, tables, ln)]
        outs = []
        for _ in range(25):
            out = torch.empty(q.shape, device=DEV)
            if window:
                compute.batched_paged_attention_decode_window(*held, out, len(lens), hq, hkv, d, 16, tables.shape[1], d ** -0.5, window, sinks, num_blocks=blocks)
            else:
                compute.batched_paged_attention_decode(*held, out, len(lens), hq, hkv, d, 16, tables.shape[1], d ** -0.5, num_blocks=blocks)
            outs.append(out)
        compute.sync()
        R.assert_close(outs[0].cpu().numpy(), want, bound, what=f"{hq}/{hkv}/{d} {window}")
        assert all(torch.equal(outs[0], o) for o in outs[1:])


@pytest.mark.gpu
def test_window_calls_replay_from_a_graph():
    import torch
    import granite_b200 as g
    side = torch.cuda.Stream(device=DEV)
    o = g.CudaCompute(0, side.cuda_stream)
    q, k, v, tables, lens, blocks, want, bound = _decode_case(8, [500, 3000, 40], 32, 8, 128, 256, 4)
    held = [_dev(x) for x in (q, k, v, tables, lens)]
    out = torch.zeros(q.shape, device=DEV)
    rng = np.random.default_rng(1)
    pk, pv = _cache(rng, 8, 400, 128)
    pq = rng.standard_normal((400, 32, 128), dtype=np.float32)
    pd = [_dev(x) for x in (pq, pk, pv)]
    p_out = torch.zeros(pq.shape, device=DEV)
    p_want, p_bound = R.attend(pq.astype(np.float64), pk.transpose(1, 0, 2).astype(np.float64), pv.transpose(1, 0, 2).astype(np.float64), np.arange(400), 128 ** -0.5, 100, 4)

    def calls():
        o.batched_paged_attention_decode_window(*held, out, 3, 32, 8, 128, 16, tables.shape[1], 128 ** -0.5, 256, 4, num_blocks=blocks)
        o.multihead_attention_window(*pd, p_out, 32, 8, 400, 400, 128, 128 ** -0.5, 100, 4)

    torch.cuda.synchronize()
    calls()
    o.sync()
    out.zero_(), p_out.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        calls()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    o.sync()
    R.assert_close(out.cpu().numpy(), want, bound, what="decode replay")
    R.assert_close(p_out.cpu().numpy(), p_want, p_bound, what="prefill replay")
    del graph
    o.shutdown()


# --------------------------------------------------------------------------------------------- refusals (no device needed)
SHARED = [(dict(window=0), "InvalidArgument", "window"), (dict(window=None), "NullPointer", "window"), (dict(q=None), "NullPointer", "null"),
          (dict(num_heads=5), "InvalidArgument", "multiple"), (dict(head_dim=100), "InvalidArgument", "head_dim"), (dict(q=264), "InvalidArgument", "aligned"),
          (dict(output=260), "InvalidArgument", "aligned"), (dict(), "NullPointer", "compute object")]


def _window(kw):
    from granite_b200 import capi
    w = kw.get("window", 8)
    return None if w is None else C.byref(capi.AttentionWindow(w, 2))


@pytest.mark.parametrize("kw,code,word", SHARED + [(dict(block_tables=None), "NullPointer", "null"), (dict(num_blocks=0), "InvalidArgument", "empty")])
def test_decode_window_refusals(kw, code, word):
    from granite_b200 import capi
    a = dict(q=256, k_cache=256, v_cache=256, block_tables=256, seq_lens=256, output=256, batch_size=1, num_heads=4, num_kv_heads=2, head_dim=128,
             block_size=16, max_blocks_per_seq=4, num_blocks=4, scale=0.1)
    a.update({k: v for k, v in kw.items() if k in a})
    got, text = _refusal(capi.lib.granite_cuda_batched_paged_attention_decode_window, C.byref(capi.PagedDecodeArgs(**a)), _window(kw))
    assert got.name == code and word in text


@pytest.mark.parametrize("seq_q", [1, 7])
@pytest.mark.parametrize("kw,code,word", SHARED + [(dict(k=None), "NullPointer", "null"), (dict(seq_kv=9, max_seq=8), "InvalidArgument", "max_seq"),
                                                   (dict(seq_kv=0), "InvalidArgument", "max_seq"), (dict(q_dtype=2), "InvalidArgument", "")])
def test_multihead_window_refusals(kw, code, word, seq_q):
    from granite_b200 import capi
    a = dict(q=256, k=256, v=256, output=256, num_heads=4, num_kv_heads=2, seq_q=seq_q, seq_kv=8, head_dim=128, scale=0.1)
    a.update({k: v for k, v in kw.items() if k != "window"})
    got, text = _refusal(capi.lib.granite_cuda_multihead_attention_window, C.byref(capi.AttentionArgs(**a)), _window(kw))
    assert got.name == code and word in text


def test_prefill_window_positions_stay_in_range():
    from granite_b200 import capi
    a = dict(q=256, k=256, v=256, output=256, num_heads=4, num_kv_heads=2, seq_q=8, seq_kv=8, head_dim=128, start_pos=0x7ffffffc, scale=0.1)
    got, text = _refusal(capi.lib.granite_cuda_multihead_attention_window, C.byref(capi.AttentionArgs(**a)), _window({}))
    assert got.name == "InvalidArgument" and "2^31" in text


@pytest.mark.parametrize("kw,code,word", SHARED + [(dict(block_table=None), "NullPointer", "null"), (dict(start_pos=61), "InvalidArgument", "beyond")])
def test_paged_prefill_window_refusals(kw, code, word):
    from granite_b200 import capi
    a = dict(q=256, k_cache=256, v_cache=256, block_table=256, output=256, num_heads=4, num_kv_heads=2, seq_q=4, start_pos=0, head_dim=128, block_size=16,
             max_blocks_per_seq=4, num_blocks=4, scale=0.1)
    a.update({k: v for k, v in kw.items() if k in a})
    got, text = _refusal(capi.lib.granite_cuda_paged_prefill_attention_window, C.byref(capi.PagedPrefillArgs(**a)), _window(kw))
    assert got.name == code and word in text
