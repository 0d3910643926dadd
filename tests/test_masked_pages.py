"""Decode over pages most of which have rows that the query does not see: every such page is cleared in its ring slot before it is
multiplied, and the slot is copied into again right after.  Repeated runs give the same bits, and the right ones."""
import numpy as np
import pytest

import view_reference as R
from test_q8_cache import _dev
from test_sliding_window import _decode_case

DEV = "cuda:0"


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (64, 8, 64), (8, 8, 128), (16, 2, 128), (96, 8, 128)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (9, 3), (40, 21)])
def test_slots_of_masked_pages_are_reused_in_order(compute, hq, hkv, d, window, sinks):
    import torch
    lens = [33, 7, 61, 1, 17, 250, 49, 100] * 40  # ragged ends everywhere; the ring wraps many times in every CTA
    q, k, v, tables, ln, blocks, want, bound = _decode_case(d + window, lens, hq, hkv, d, window, sinks)
    held = [_dev(x) for x in (q, k, v, tables, ln)]
    outs = []
    for _ in range(30):
        out = torch.full(q.shape, float("nan"), device=DEV)
        if window:
            compute.batched_paged_attention_decode_window(*held, out, len(lens), hq, hkv, d, 16, tables.shape[1], d ** -0.5, window, sinks, num_blocks=blocks)
        else:
            compute.batched_paged_attention_decode(*held, out, len(lens), hq, hkv, d, 16, tables.shape[1], d ** -0.5, num_blocks=blocks)
        outs.append(out)
    compute.sync()
    R.assert_close(outs[0].cpu().numpy(), want, bound, what=f"{hq}/{hkv}/{d} {window}+{sinks}")
    assert all(torch.equal(outs[0], o) for o in outs[1:])
