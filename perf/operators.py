"""The operators around an 8-bit paged K/V cache and a sliding window, as one pass each.

Five operators of the attention path:

  append_q8       rotate Q and K of new tokens, write K and V into the paged cache in 8 bits with one fp32
                  scale per (page, KV head); a page whose scale grows has its older rows re-coded
  decode_q8       one query token per sequence over that cache, optionally with a sliding window and sinks
  prefill_q8      a chunk of query tokens of one sequence over that cache
  decode_window   one query token per sequence over the fp16 cache: the last `window` keys and the first
                  `sinks` keys are visible
  prefill_window  causal prefill with the same visibility rule, contiguous or paged fp16 cache

Layouts: pools [num_blocks * block_size, Hkv, D], scales [num_blocks, Hkv], tables [B, max_blocks] int32,
queries [B, Hq, D] (decode) or [S, Hq, D] (prefill).  An 8-bit code stands for code * scale; codes are int8
in [-127, 127] or fp8 e4m3 in [-448, 448].
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
INT8, E4M3 = 0, 1
QMAX = (127.0, 448.0)


# ------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of 64 running sequences writes its tokens (latency)
        dict(name="append step e4m3 b64", op="append_q8", dtype="e4m3", batch=64, new_len=1, lo=1024, hi=32768, hq=32, hkv=8, d=128),
        # five accepted draft tokens for each of 16 sequences, pages ending inside the run
        dict(name="append draft int8 b16 d64", op="append_q8", dtype="int8", batch=16, new_len=5, lo=1, hi=5000, hq=32, hkv=8, d=64),
        # prompt chunks of four sequences enter the cache
        dict(name="append chunk e4m3 4x2043", op="append_q8", dtype="e4m3", batch=4, new_len=2043, lo=0, hi=9000, hq=32, hkv=8, d=128),
        # a single user's step over a short context (latency)
        dict(name="decode int8 b1 ctx512", op="decode_q8", dtype="int8", batch=1, lo=512, hi=512, hq=32, hkv=8, d=128, window=0, sinks=0),
        # a serving batch of ragged contexts (bandwidth)
        dict(name="decode e4m3 b64 32k", op="decode_q8", dtype="e4m3", batch=64, lo=1024, hi=32768, hq=32, hkv=8, d=128, window=0, sinks=0),
        # many sequences whose visible keys are a window of 4096 and four sinks
        dict(name="decode int8 b96 window4096", op="decode_q8", dtype="int8", batch=96, lo=100, hi=20000, hq=64, hkv=8, d=128, window=4096, sinks=4),
        # a single user's step of a windowed layer over the fp16 cache (latency)
        dict(name="window decode b1 8191", op="decode_window", paged=False, batch=1, lo=8191, hi=8191, hq=32, hkv=8, d=128, window=1024, sinks=4),
        # a serving batch of a windowed layer (bandwidth)
        dict(name="window decode b64 32k", op="decode_window", paged=True, batch=64, lo=1024, hi=32768, hq=32, hkv=8, d=128, window=4096, sinks=20),
        # a whole prompt of a windowed layer
        dict(name="window prefill 2048", op="prefill_window", paged=False, seq=2048, start=0, hq=32, hkv=8, d=128, window=512, sinks=0, half=True),
        # a late chunk of a long prompt over the paged cache, fp32 queries and outputs
        dict(name="window prefill 4001@4099", op="prefill_window", paged=True, seq=4001, start=4099, hq=32, hkv=8, d=128, window=2047, sinks=4, half=False),
        # a short chunk over a short 8-bit context
        dict(name="prefill e4m3 509@1531", op="prefill_q8", dtype="e4m3", seq=509, start=1531, hq=32, hkv=8, d=128, window=0, sinks=0, half=False),
        # a full chunk deep in a prompt
        dict(name="prefill int8 2048@14336", op="prefill_q8", dtype="int8", seq=2048, start=14336, hq=32, hkv=8, d=128, window=0, sinks=0, half=True),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["append_q8", "decode_q8", "prefill_q8", "decode_window", "prefill_window"])
    hkv = rng.choice([1, 2, 4, 8])
    case = dict(op=op, hq=hkv * rng.choice([1, 2, 4, 8]), hkv=hkv, d=rng.choice([64, 128, 128]))
    if op in ("append_q8", "decode_q8", "prefill_q8"):
        case["dtype"] = rng.choice(["int8", "e4m3"])
    if op == "append_q8":
        case["batch"] = log(1, 128)
        case["new_len"] = log(1, max(2, 8192 // case["batch"]))
        case["lo"], case["hi"] = 0, log(16, 32000)
        return case
    if op in ("decode_q8", "decode_window"):
        case["batch"] = log(1, 64)
        case["hi"] = log(16, 32768)
        case["lo"] = rng.randint(1, case["hi"])
    else:
        case["seq"] = log(2, 2048)
        case["start"] = rng.choice([0, log(1, 4096)])
        case["half"] = rng.random() < 0.5
    windowed = op in ("decode_window", "prefill_window") or rng.random() < 0.5
    case["window"] = log(16, 8192) if windowed else 0
    case["sinks"] = rng.choice([0, rng.randint(1, 40)]) if windowed else 0
    if op in ("decode_window", "prefill_window"):
        case["paged"] = rng.random() < 0.5
    if op == "decode_window" and not case["paged"]:
        case["lo"] = case["hi"]  # the contiguous call has one length for the batch
    return case


# ------------------------------------------------------------------------------------------- inputs
PAGE = 16


def _positions(case, seed):
    """Lengths (or write positions) of the sequences, from the seed."""
    r = np.random.default_rng(seed)
    return r.integers(case["lo"], case["hi"] + 1, size=case["batch"]).astype(np.int32)


def _tables(first, last, seed, num=0):
    """Block tables that map the logical pages [first, last) of each sequence to a random permutation of
    the pool's pages (at least `num`); entries before them are -1 (never looked at)."""
    counts = (last - first).astype(np.int64)
    num = max(int(counts.sum()), num, 1)
    perm = np.random.default_rng(seed + 100).permutation(num).astype(np.int32)
    tables = np.full((len(first), max(int(last.max()), 1)), -1, np.int32)
    off = 0
    for b in range(len(first)):
        tables[b, first[b]:last[b]] = perm[off:off + counts[b]]
        off += int(counts[b])
    return tables, num


def _codes(gen, rows, hkv, d, dtype):
    """A pool of codes as a cache holds them: values near N(0, 1) over a page whose largest is the code range's end."""
    x = torch.empty((rows, hkv, d), dtype=torch.float16, device=DEV).normal_(generator=gen)
    if dtype == "int8":
        return x.mul_(32.0).round_().clamp_(-127, 127).to(torch.int8)
    return x.mul_(112.0).clamp_(-448, 448).to(torch.float8_e4m3fn)


def _rope_tables(n, d):
    inv = torch.pow(10000.0, -torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d)
    a = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] * inv
    return a.cos().float(), a.sin().float()


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    s = dict(case=case, scale=1.0 / math.sqrt(d))

    def normal(*shape):
        return torch.empty(shape, device=DEV).normal_(generator=gen)

    def scales(blocks, dtype):
        return (0.5 + torch.rand((blocks, hkv), device=DEV, generator=gen)) / (32.0 if dtype == "int8" else 112.0)

    if case["op"] == "append_q8":
        pos = _positions(case, seed)
        first, last = pos // PAGE, (pos + case["new_len"] + PAGE - 1) // PAGE
        tables, blocks = _tables(first, last, seed, case["batch"] * ((case["new_len"] + 2 * PAGE - 2) // PAGE))
        s["cos"], s["sin"] = _rope_tables(int((pos + case["new_len"]).max()), d)
        s["q"] = normal(case["batch"], case["new_len"], hq, d)
        s["k"], s["v"] = normal(case["batch"], case["new_len"], hkv, d), normal(case["batch"], case["new_len"], hkv, d)
        s["lens"] = torch.from_numpy(pos).to(DEV)
    elif case["op"] in ("decode_q8", "decode_window"):
        lens = _positions(case, seed)
        tables, blocks = _tables(np.zeros_like(lens), (lens + PAGE - 1) // PAGE, seed)
        s["q"] = normal(case["batch"], hq, d)
        s["lens"] = torch.from_numpy(lens).to(DEV)
        s["len"] = int(lens[0])
        s["out"] = torch.empty((case["batch"], hq, d), device=DEV)
    else:
        end = case["start"] + case["seq"]
        tables, blocks = _tables(np.zeros(1, np.int32), np.array([(end + PAGE - 1) // PAGE], np.int32), seed)
        s["q"] = normal(case["seq"], hq, d)
        if case["half"]:
            s["q"] = s["q"].half()
        s["out"] = torch.empty_like(s["q"])
    s["tables"], s["blocks"] = torch.from_numpy(tables).to(DEV), blocks
    if "dtype" in case:
        s["k_cache"], s["v_cache"] = (_codes(gen, blocks * PAGE, hkv, d, case["dtype"]) for _ in range(2))
        s["k_scales"], s["v_scales"] = scales(blocks, case["dtype"]), scales(blocks, case["dtype"])
    elif case["paged"]:
        s["k_cache"], s["v_cache"] = normal(blocks * PAGE, hkv, d).half(), normal(blocks * PAGE, hkv, d).half()
    else:
        n = s["len"] if case["op"] == "decode_window" else case["start"] + case["seq"]
        b = case.get("batch", 1)
        s["k_cache"], s["v_cache"] = normal(b, hkv, n, d).half(), normal(b, hkv, n, d).half()
    return s


# ------------------------------------------------------------------------------------------- plain form
def _rotate(x, cos, sin):
    """Adjacent pairs rotated; cos and sin [..., 1, D/2] broadcast over the heads."""
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)


def _encode(x, dtype):
    return x.round().clamp(-127, 127).to(torch.int8) if dtype == "int8" else x.to(torch.float8_e4m3fn)


def _append_plain(s):
    case = s["case"]
    n, qmax = case["new_len"], QMAX[0] if case["dtype"] == "int8" else QMAX[1]
    where = s["lens"].long()[:, None] + torch.arange(n, device=DEV)          # [B, n] positions
    cos, sin = s["cos"][where][:, :, None], s["sin"][where][:, :, None]
    s["q"].copy_(_rotate(s["q"], cos, sin))
    # slot j of touched page p holds new token p * PAGE + j - off
    off = s["lens"].long() % PAGE
    pages = (n + PAGE - 1) // PAGE + 1
    slot = torch.arange(pages * PAGE, device=DEV).view(1, pages, PAGE)
    token = slot - off[:, None, None]
    new, old = (token >= 0) & (token < n), token < 0                          # [B, pages, PAGE]
    touched = new.any(-1)
    logical = (s["lens"].long() // PAGE)[:, None] + torch.arange(pages, device=DEV)
    phys = s["tables"].long().gather(1, logical.clamp(max=s["tables"].shape[1] - 1))[touched]  # [T]
    seq = torch.arange(case["batch"], device=DEV)[:, None].expand(-1, pages)[touched]
    token, new, old = token[touched].clamp(0, n - 1), new[touched][..., None, None], old[touched][..., None, None]
    for x, cache, scales in ((_rotate(s["k"], cos, sin), s["k_cache"], s["k_scales"]), (s["v"], s["v_cache"], s["v_scales"])):
        x = x[seq[:, None], token]                                            # [T, PAGE, Hkv, D]
        need = (x.abs() * new).amax((1, 3)) / qmax                            # [T, Hkv]
        before = torch.where(old.any(1)[..., 0], scales[phys], 0.0)
        after = torch.maximum(before, need)
        unit = torch.where(after > 0, after, 1.0)
        rows = cache.view(-1, PAGE, *cache.shape[1:])
        codes = rows[phys].float()
        moved = _encode(codes * (before / unit)[:, None, :, None], case["dtype"]).float()
        fresh = _encode(x / unit[:, None, :, None], case["dtype"]).float()
        codes = torch.where(new, fresh, torch.where(old, moved, codes)).to(cache.dtype)
        rows.view(torch.uint8)[phys] = codes.view(torch.uint8)
        scales[phys] = after
    return _append_outputs(s)


def _append_outputs(s):
    """The state that an append updates.  fp8 codes are values already; int8 ones are given as the values they stand for."""
    k, v = s["k_cache"], s["v_cache"]
    if s["case"]["dtype"] == "int8":
        k, v = ((c.view(-1, PAGE, *c.shape[1:]) * f[:, None, :, None]).half() for c, f in ((k, s["k_scales"]), (v, s["v_scales"])))
    return {"q": s["q"], "k": k, "v": v, "k_scales": s["k_scales"], "v_scales": s["v_scales"]}


def _paged_rows(s, which):
    """Cache rows of every sequence in order, in 32 bits: [B, max_blocks * PAGE, Hkv, D]."""
    t = s["tables"].long().clamp(min=0)
    x = s[which + "_cache"].view(-1, PAGE, *s[which + "_cache"].shape[1:])
    x = (x.view(torch.uint8)[t].view(x.dtype) if x.element_size() == 1 else x[t]).float()
    if which + "_scales" in s:
        x = x * s[which + "_scales"][t][:, :, None, :, None]
    return x.flatten(1, 2)


def _cache_rows(s):
    if s["case"].get("paged", True):
        return _paged_rows(s, "k").transpose(1, 2), _paged_rows(s, "v").transpose(1, 2)
    return s["k_cache"].float(), s["v_cache"].float()


def _softmax_attend(q, k, v, visible, scale):
    """q [B, Hkv, R, D], k and v [B, Hkv, N, D], visible broadcast to [B, Hkv, R, N]."""
    x = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).masked_fill_(~visible, -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True)).exp_()
    return torch.matmul(x, v) / x.sum(-1, keepdim=True)


def _visible(pos, key, window, sinks):
    seen = key <= pos
    return seen & ((pos - key < window) | (key < sinks)) if window else seen


def _decode_plain(s):
    case = s["case"]
    k, v = _cache_rows(s)
    q = s["q"].view(case["batch"], case["hkv"], -1, case["d"])
    last = s["lens"].long().view(-1, 1, 1, 1) - 1
    visible = _visible(last, torch.arange(k.shape[2], device=DEV), case["window"], case["sinks"])
    return _softmax_attend(q, k, v, visible, s["scale"]).reshape(s["q"].shape)


def _prefill_plain(s):
    case = s["case"]
    k, v = _cache_rows(s)
    n, g = case["seq"], case["hq"] // case["hkv"]
    q = s["q"].float().view(n, case["hkv"], g, case["d"]).permute(1, 2, 0, 3).reshape(1, case["hkv"], g * n, case["d"])
    pos = case["start"] + torch.arange(n, device=DEV).repeat(g)[:, None]
    o = _softmax_attend(q, k, v, _visible(pos, torch.arange(k.shape[2], device=DEV), case["window"], case["sinks"]), s["scale"])
    o = o.view(case["hkv"], g, n, case["d"]).permute(2, 0, 1, 3).reshape(n, case["hq"], case["d"])
    return o.to(s["q"].dtype)


# ------------------------------------------------------------------------------------------- the framework's calls
_objects = {}


def _compute():
    """The program's compute object for the current device and stream."""
    import granite_b200
    key = (torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream)
    if key not in _objects:
        _objects[key] = granite_b200.CudaCompute(*key)
    return _objects[key]


def _run_own(s):
    case, c = s["case"], _compute()
    op, hq, hkv, d = case["op"], case["hq"], case["hkv"], case["d"]
    code = E4M3 if case.get("dtype") == "e4m3" else INT8
    blocks, width = s["blocks"], s["tables"].shape[1]
    if op == "append_q8":
        c.rope_paged_kv_cache_append_q8(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["k_cache"], s["v_cache"], s["k_scales"],
                                        s["v_scales"], s["tables"], s["lens"], case["batch"], case["new_len"], hq, hkv, d,
                                        PAGE, width, blocks, s["cos"].shape[0], code)
        return _append_outputs(s)
    if op == "decode_q8":
        c.batched_paged_attention_decode_q8(s["q"], s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"], s["tables"],
                                            s["lens"], s["out"], case["batch"], hq, hkv, d, PAGE, width, s["scale"],
                                            num_blocks=blocks, cache_dtype=code, window=case["window"], sinks=case["sinks"])
    elif op == "prefill_q8":
        half = int(case["half"])
        c.paged_prefill_attention_q8(s["q"], s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"], s["tables"], s["out"],
                                     hq, hkv, case["seq"], case["start"], d, PAGE, width, blocks, s["scale"], code,
                                     q_dtype=half, out_dtype=half, window=case["window"], sinks=case["sinks"])
    elif op == "decode_window":
        if case["paged"]:
            c.batched_paged_attention_decode_window(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["lens"], s["out"],
                                                    case["batch"], hq, hkv, d, PAGE, width, s["scale"], case["window"],
                                                    case["sinks"], num_blocks=blocks)
        else:
            c.multihead_attention_window(s["q"], s["k_cache"], s["v_cache"], s["out"], hq, hkv, 1, s["len"], d, s["scale"],
                                         case["window"], case["sinks"], batch_size=case["batch"])
    else:
        half, end = int(case["half"]), case["start"] + case["seq"]
        if case["paged"]:
            c.paged_prefill_attention_window(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["out"], hq, hkv, case["seq"],
                                             case["start"], d, PAGE, width, blocks, s["scale"], case["window"], case["sinks"],
                                             q_dtype=half, out_dtype=half)
        else:
            c.multihead_attention_window(s["q"], s["k_cache"], s["v_cache"], s["out"], hq, hkv, case["seq"], end, d, s["scale"],
                                         case["window"], case["sinks"], q_dtype=half, out_dtype=half, start_pos=case["start"])
    return s["out"]


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "append_q8":
        return _append_plain(state)
    return _decode_plain(state) if op.startswith("decode") else _prefill_plain(state)


# ------------------------------------------------------------------------------------------- what a pass cannot do without
def _seen(pos, window, sinks):
    """Keys that a query at position `pos` (array) sees."""
    pos = np.asarray(pos, np.float64)
    return np.minimum(pos + 1, window + np.minimum(sinks, np.maximum(pos + 1 - window, 0))) if window else pos + 1


def work(case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    bytes_per = 1 if "dtype" in case else 2
    if case["op"] == "append_q8":
        tokens = case["batch"] * case["new_len"]
        rows = tokens * hkv * d
        # Q read and written, K and V read in 32 bits and written in 8, a scale per page and head read and written, the angles
        b = tokens * hq * d * 8 + rows * 2 * 5 + (tokens / PAGE + case["batch"]) * hkv * 2 * 8 + tokens * d * 4
        return {"bytes": b, "flops": tokens * (hq + hkv) * d * 3 + rows * 2 * 3}
    row = hkv * d * bytes_per * 2 + (hkv * 8 / PAGE if "dtype" in case else 0)   # K and V of one token, its share of the scales
    if "batch" in case:
        mid = np.linspace(case["lo"], case["hi"], 257) - 1
        keys = case["batch"] * float(_seen(mid, case["window"], case["sinks"]).mean())
        return {"bytes": keys * row + case["batch"] * hq * d * 8, "flops": keys * hq * d * 4}
    n, start = case["seq"], case["start"]
    pairs = float(_seen(start + np.arange(n), case["window"], case["sinks"]).sum())
    far = min(start + n, (case["window"] + n - 1 + case["sinks"]) if case["window"] else start + n)
    return {"bytes": far * row + n * hq * d * (4 if case["half"] else 8), "flops": pairs * hq * d * 4}


# ------------------------------------------------------------------------------------------- in 64 bits, from the definitions
def _round_e4m3(x):
    """Nearest e4m3 value, ties to even: steps of 2^(e-3) for 2^e <= |x| < 2^(e+1), 2^-9 below 2^-6."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))).clamp(max=8)
    e = torch.where(torch.exp2(e) > x.abs().clamp(min=2.0 ** -6), e - 1, e)
    step = torch.exp2(e - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_append(s):
    case = s["case"]
    n, int8 = case["new_len"], case["dtype"] == "int8"
    near = (lambda x: torch.round(x).clamp(-127, 127)) if int8 else _round_e4m3
    out = {"q": s["q"].double(), "k": s["k_cache"].double(), "v": s["v_cache"].double(),
           "k_scales": s["k_scales"].double(), "v_scales": s["v_scales"].double()}
    pos, tables = s["lens"].tolist(), s["tables"].cpu()
    for b in range(case["batch"]):
        c, si = (s[t][pos[b]:pos[b] + n].double()[:, None] for t in ("cos", "sin"))
        turned = {}
        for name in ("q", "k"):
            pair = torch.view_as_complex(s[name][b].double().unflatten(-1, (-1, 2)).contiguous()) * torch.complex(c, si)
            turned[name] = torch.view_as_real(pair).flatten(-2)
        out["q"][b] = turned["q"]
        for name, x in (("k", turned["k"]), ("v", s["v"][b].double())):
            at = pos[b]
            while at < pos[b] + n:
                end = min((at // PAGE + 1) * PAGE, pos[b] + n)
                page, j = int(tables[b, at // PAGE]), at % PAGE
                rows = x[at - pos[b]:end - pos[b]]
                had = out[name + "_scales"][page] * (1.0 if j else 0.0)
                now = torch.maximum(had, rows.abs().amax((0, 2)) / (127.0 if int8 else 448.0))
                codes = out[name][page * PAGE:(page + 1) * PAGE]
                codes[:j] = near(codes[:j] * (had / now)[:, None])
                codes[j:j + end - at] = near(rows / now[:, None])
                out[name + "_scales"][page] = now
                at = end
    if int8:
        for name in ("k", "v"):
            out[name] = out[name].view(-1, PAGE, case["hkv"], case["d"]) * out[name + "_scales"][:, None, :, None]
    return out


def _exact_rows(s, which, b, n):
    """[Hkv, n, D] rows of sequence b in 64 bits."""
    if not s["case"].get("paged", True):
        return s[which + "_cache"][b, :, :n].double()
    p = torch.arange(n, device=DEV)
    page = s["tables"][b].long()[p // PAGE]
    codes = s[which + "_cache"]
    at = page * PAGE + p % PAGE
    x = (codes.view(torch.uint8)[at].view(codes.dtype) if codes.element_size() == 1 else codes[at]).double()
    if which + "_scales" in s:
        x = x * s[which + "_scales"].double()[page][:, :, None]
    return x.transpose(0, 1)


def _exact_heads(q, k, v, hidden, scale):
    """q [R, D] against k, v [n, D]; hidden [R, n]."""
    x = (q @ k.T) * scale
    x[hidden] = -math.inf
    return torch.softmax(x, -1) @ v


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append_q8":
        return _exact_append(s)
    g, w, sinks = case["hq"] // case["hkv"], case["window"], case["sinks"]
    q = s["q"].double()
    out = torch.empty_like(q)
    if "batch" in case:
        for b, n in enumerate(s["lens"].tolist()):
            k, v = _exact_rows(s, "k", b, n), _exact_rows(s, "v", b, n)
            j = torch.arange(n, device=DEV)
            hidden = (j < n - w) & (j >= sinks) if w else j < 0
            for h in range(case["hkv"]):
                out[b, h * g:(h + 1) * g] = _exact_heads(q[b, h * g:(h + 1) * g], k[h], v[h], hidden.expand(g, n), s["scale"])
        return out
    n = case["start"] + case["seq"]
    k, v = _exact_rows(s, "k", 0, n), _exact_rows(s, "v", 0, n)
    i, j = torch.arange(case["start"], n, device=DEV)[:, None], torch.arange(n, device=DEV)
    hidden = j > i
    if w:
        hidden = hidden | ((j <= i - w) & (j >= sinks))
    for h in range(case["hq"]):
        out[:, h] = _exact_heads(q[:, h], k[h // g], v[h // g], hidden, s["scale"])
    return out
