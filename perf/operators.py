"""Attention over packed sequences, its gradient, the paged key/value cache and the attention that reads it, as measurable cases.

Each case is one call of one operator on buffers that a program keeps on the GPU:

  fwd    attention over a whole prompt: sequences of different lengths packed row after row, grouped heads, causal or not
  grad   its gradients with respect to q, k and v, from the forward's output and log-sum-exp
  write  the new tokens' keys and values into a paged cache, as they are or as e4m3 with one power-of-two scale per row
  read   a cache's keys and values back into packed rows
  paged  attention of each sequence's new tokens over its cached keys and values

`own` false: elementary torch operations in 32 bits, rounded once at the end. `own` true: the kernel library's entry points.
Lengths are texts ("512,64"), so that a case is plain values.
"""
import math
import os
import sys

import torch

own = False

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if os.path.join(REPO, "frame-public_amd") not in sys.path:
    sys.path.insert(0, os.path.join(REPO, "frame-public_amd"))

TORCH = {"bf16": torch.bfloat16, "f16": torch.float16}


# ---- the cases --------------------------------------------------------------------------------------------------

def listed():
    return [
        # a server's smallest prefill: a few short prompts, one empty and one of a single token; launches and latency
        dict(name="fwd_short", kind="fwd", dtype="f16", heads=8, kv_heads=2, dh=64, lens="1,17,64,129,5,0,200", pad=3,
             causal=True, fused=True),
        # the transformer block's attention (16 heads of 64) with its batch of eight sequences packed and masked
        dict(name="fwd_block", kind="fwd", dtype="bf16", heads=16, kv_heads=16, dh=64, lens="512,512,512,512,512,512,512,512",
             pad=0, causal=True, fused=False),
        # long prompts of a model with grouped heads; q, k and v are columns of one projection's output
        dict(name="fwd_long", kind="fwd", dtype="bf16", heads=32, kv_heads=8, dh=128, lens="5003,2318,871", pad=0,
             causal=True, fused=True),
        # a training step's backward at the block's sizes, lengths as a packed batch has them
        dict(name="grad_block", kind="grad", dtype="bf16", heads=16, kv_heads=16, dh=64,
             lens="512,384,301,512,77,512,490,512", pad=6, causal=True, fused=False),
        # a long-context training step with grouped heads
        dict(name="grad_long", kind="grad", dtype="bf16", heads=32, kv_heads=8, dh=128, lens="2897,1034,165", pad=0,
             causal=True, fused=True),
        # one decoding step of 64 sequences: a row each, quantised as it is written
        dict(name="write_step", kind="write", dtype="bf16", cache="e4m3", kv_heads=8, dh=128, page=16,
             new=_same(64, 1), past=_steps(64, 100, 97), pad=0),
        # a prefill's keys and values
        dict(name="write_prompt", kind="write", dtype="bf16", cache="e4m3", kv_heads=8, dh=128, page=64,
             new="5003,2318,871", past="0,0,1000", pad=0),
        # a few short sequences from an unquantised cache
        dict(name="read_short", kind="read", dtype="f16", cache="f16", kv_heads=4, dh=64, page=16, lens="1,130,77,1000"),
        # a batch's whole context, as a prefix that is computed on again or moved
        dict(name="read_long", kind="read", dtype="bf16", cache="e4m3", kv_heads=8, dh=128, page=64,
             lens="16384,9001,8192,12345,2048,777,4096,12693"),
        # one sequence with a long context, one new token: nothing but the cache's bytes and the latency
        dict(name="paged_one", kind="paged", dtype="bf16", cache="bf16", heads=32, kv_heads=8, dh=128, page=16, new="1",
             past="32767", pad=0),
        # a serving batch's decoding step over a quantised cache
        dict(name="paged_batch", kind="paged", dtype="bf16", cache="e4m3", heads=32, kv_heads=8, dh=128, page=64,
             new=_same(64, 1), past=_steps(64, 127, 128), pad=0),
        # chunks of prompts whose beginnings are cached, next to sequences that decode
        dict(name="paged_chunk", kind="paged", dtype="bf16", cache="bf16", heads=32, kv_heads=8, dh=128, page=64,
             new="512,509,1,300,512,1,190", past="4096,7683,2200,0,1536,900,5555", pad=8),
    ]


def _same(n, value):
    return ",".join([str(value)] * n)


def _steps(n, first, step):
    return ",".join(str(first + i * step) for i in range(n))


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _lens(rng, most_seqs, longest, total):
    """Lengths of up to most_seqs sequences, spread over their logarithm, whose sum stays within `total`."""
    out = []
    for _ in range(_log_int(rng, 1, most_seqs)):
        n = _log_int(rng, 1, longest)
        if sum(out) + n > total:
            break
        out.append(n)
    return out or [_log_int(rng, 1, longest)]


def _heads(rng):
    kv_heads = rng.choice([1, 2, 4, 8, 5])
    return kv_heads * rng.choice([1, 2, 3, 4, 8]), kv_heads


def draw(rng):
    """One case of the ranges above: lengths over their logarithm, any number of tokens, heads in groups of one to eight."""
    kind = rng.choice(["fwd", "fwd", "grad", "grad", "write", "read", "paged", "paged", "paged"])
    heads, kv_heads = _heads(rng)
    dtype = rng.choice(["bf16", "bf16", "f16"])
    dh = rng.choice([64, 64, 128, 128, 96, 80, 32])
    if kind in ("fwd", "grad"):
        while True:
            lens = _lens(rng, 24, 4096 if kind == "fwd" else 2048, 6144)
            if heads * dh * sum(n * n for n in lens) <= 2 ** 34:
                return dict(kind=kind, dtype=dtype, heads=heads, kv_heads=kv_heads, dh=dh, lens=_text(lens),
                            pad=rng.choice([0, 0, 5]), causal=rng.random() < 0.75, fused=rng.random() < 0.5)
            heads = kv_heads
    cache, page = rng.choice([dtype, "e4m3"]), rng.choice([8, 16, 32, 64, 128, 256])
    if kind == "read":
        return dict(kind=kind, dtype=dtype, cache=cache, kv_heads=kv_heads, dh=dh, page=page,
                    lens=_text(_lens(rng, 64, 16384, 32768)))
    if kind == "write":
        new = _lens(rng, 64, rng.choice([1, 16, 4096]), 8192)
        return dict(kind=kind, dtype=dtype, cache=cache, kv_heads=kv_heads, dh=dh, page=page, new=_text(new),
                    past=_text([rng.choice([0, _log_int(rng, 1, 4096)]) for _ in new]), pad=rng.choice([0, 0, 5]))
    while True:
        new = _lens(rng, 64, rng.choice([1, 1, 8, 700]), 2048)
        past = [rng.choice([0, _log_int(rng, 1, 16384), _log_int(rng, 1, 16384)]) for _ in new]
        pairs = sum(n * (n + p) for n, p in zip(new, past))
        # the plain form's score tensor is new x cached of the longest ones
        if max(new) * max(n + p for n, p in zip(new, past)) * len(new) * heads <= 2 ** 31 and heads * dh * pairs <= 2 ** 33 \
                and sum(past) * kv_heads * dh <= 2 ** 28 and max(past) * len(new) * kv_heads * dh <= 2 ** 30:
            return dict(kind=kind, dtype=dtype, cache=cache, heads=heads, kv_heads=kv_heads, dh=dh, page=page,
                        new=_text(new), past=_text(past), pad=rng.choice([0, 0, 5]))


def _text(lens):
    return ",".join(str(n) for n in lens)


def _ints(text):
    return [int(n) for n in text.split(",")]


# ---- work -------------------------------------------------------------------------------------------------------

def _pairs(case):
    """Query-key pairs of one head that the mask leaves."""
    if case["kind"] == "paged":
        return sum(n * p + n * (n + 1) // 2 for n, p in zip(_ints(case["new"]), _ints(case["past"])))
    return sum(n * (n + 1) // 2 if case["causal"] else n * n for n in _ints(case["lens"]))


def _cache_row(case):
    """Bytes of a cached key or value row of one head."""
    return case["dh"] + 1 if case["cache"] == "e4m3" else 2 * case["dh"]


def work(case):
    kind, dh, kv = case["kind"], case["dh"], case["kv_heads"]
    if kind in ("fwd", "grad"):
        rows, h = sum(_ints(case["lens"])), case["heads"]
        if kind == "fwd":  # q, k, v in; out and the log-sum-exp out
            return {"bytes": rows * (2 * dh * (2 * h + 2 * kv) + 4 * h), "flops": 4 * h * dh * _pairs(case)}
        # q, k, v, out, dout, log-sum-exp in; dq, dk, dv out
        return {"bytes": rows * (2 * dh * (4 * h + 4 * kv) + 4 * h), "flops": 10 * h * dh * _pairs(case)}
    if kind == "write":
        rows = sum(_ints(case["new"])) * kv * 2
        return {"bytes": rows * (2 * dh + _cache_row(case)), "flops": 0}
    if kind == "read":
        rows = sum(_ints(case["lens"])) * kv * 2
        return {"bytes": rows * (2 * dh + _cache_row(case)), "flops": 0}
    new, past, h = _ints(case["new"]), _ints(case["past"]), case["heads"]
    cached = sum(new) + sum(past)
    return {"bytes": cached * kv * 2 * _cache_row(case) + sum(new) * h * dh * 4, "flops": 4 * h * dh * _pairs(case)}


# ---- inputs -----------------------------------------------------------------------------------------------------

def _starts(lens):
    return torch.tensor([0] + list(_running(lens)), dtype=torch.int32, device="cuda")


def _running(lens):
    total = 0
    for n in lens:
        total += n
        yield total


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    s["t"] = TORCH[case["dtype"]]
    return (_prepare_packed if case["kind"] in ("fwd", "grad") else _prepare_paged)(s, g)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _prepare_packed(s, g):
    lens, h, kv, dh, t = _ints(s["lens"]), s["heads"], s["kv_heads"], s["dh"], s["t"]
    rows = sum(lens) + s["pad"]
    s.update(longest=max(lens), rows=rows, batch=len(lens), cu=_starts(lens), scale=1.0 / math.sqrt(dh))
    widths = [h * dh, kv * dh, kv * dh]

    def three():
        if s["fused"]:
            return torch.empty(rows, sum(widths), dtype=t, device="cuda").split(widths, 1)
        return [torch.empty(rows, w, dtype=t, device="cuda") for w in widths]

    s["q"], s["k"], s["v"] = three()
    for x in (s["q"], s["k"], s["v"]):
        x.copy_(_randn(g, rows, x.shape[1]))
    # what the rows behind the last sequence hold before the call, they hold after it
    s["out"] = torch.zeros(rows, h * dh, dtype=t, device="cuda")
    s["lse"] = torch.zeros(rows, h, device="cuda")
    if s["kind"] == "grad":
        out, lse = _packed_plain(s)
        s["out"].copy_(out)
        s["lse"].copy_(lse)
        s["dout"] = _randn(g, rows, h * dh).to(t)
        s["dq"], s["dk"], s["dv"] = three()
        for x in (s["dq"], s["dk"], s["dv"]):
            x.zero_()
    return s


def _prepare_paged(s, g):
    kv, dh, t, page, kind = s["kv_heads"], s["dh"], s["t"], s["page"], s["kind"]
    if kind == "read":
        cached = new = _ints(s["lens"])
    else:
        new = _ints(s["new"])
        cached = [n + p for n, p in zip(new, _ints(s["past"]))]
    used = [-(-n // page) for n in cached]
    pages, width = sum(used) + 3, max(used)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(cached), width, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    rows = sum(new) + s.get("pad", 0)
    s.update(pages=pages, table=table, rows=rows, batch=len(new), cu=_starts(new), longest_new=max(new),
             longest=max(cached), kv_lens=torch.tensor(cached, dtype=torch.int32, device="cuda"))
    shape = (pages, page, kv, dh)
    for x in "kv":
        values = _randn(g, *shape)
        if s["cache"] == "e4m3":
            s[x + "_cache"], s[x + "_scale"] = (y.contiguous() for y in _quantise(values))
        else:
            s[x + "_cache"] = values.to(t)
    if kind == "write":
        s["k"], s["v"] = (_randn(g, rows, kv * dh).to(t) for _ in "kv")
    elif kind == "read":
        s["k"], s["v"] = (torch.zeros(rows, kv * dh, dtype=t, device="cuda") for _ in "kv")
    else:
        s["q"] = _randn(g, rows, s["heads"] * dh).to(t)
        s["out"] = torch.zeros(rows, s["heads"] * dh, dtype=t, device="cuda")
        s["scale"] = 1.0 / math.sqrt(dh)
    return s


# ---- the operators in their plain form ---------------------------------------------------------------------------

def _places(cu, rows):
    """For each row the sequence it belongs to and its place in it; rows behind the last sequence: `inside` false."""
    row = torch.arange(rows, device="cuda")
    ends = cu[1:].long()
    seq = torch.searchsorted(ends, row, right=True)
    inside = seq < ends.numel()
    seq = torch.where(inside, seq, 0)
    return seq, torch.where(inside, row - cu.long()[seq], 0), inside


def _rows_of(cu, longest):
    """[batch, longest] row numbers of each sequence's places, and which of them exist."""
    place = torch.arange(longest, device="cuda")
    there = place < (cu[1:] - cu[:-1]).long()[:, None]
    return torch.where(there, cu[:-1].long()[:, None] + place, 0), there


def _grouped(x, kv, dh):
    """[batch, places, heads * dh] -> [batch, kv_heads, group * places, dh], in 32 bits."""
    b, n, width = x.shape
    return x.float().reshape(b, n, kv, width // (kv * dh), dh).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, dh)


def _ungrouped(x, n):
    """The reverse of _grouped."""
    b, kv, gn, dh = x.shape
    return x.reshape(b, kv, gn // n, n, dh).permute(0, 3, 1, 2, 4).reshape(b, n, -1)


def _probabilities(s, q, k, keys_there, limit):
    """softmax(scale * q k^T) with the keys that exist and stand at `limit` or before, and the log-sum-exp."""
    key = torch.arange(k.shape[2], device="cuda")
    seen = keys_there[:, None, :] & (key <= limit[:, :, None])               # [batch, new, keys]
    group = q.shape[2] // limit.shape[1]
    scores = (q @ k.transpose(2, 3)) * s["scale"]
    b, kv, gn, n = scores.shape
    scores = scores.reshape(b, kv, group, -1, n).masked_fill(~seen[:, None, None], -math.inf).reshape(b, kv, gn, n)
    top = scores.amax(3, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(scores - top)
    total = e.sum(3, keepdim=True)
    return e / torch.where(total == 0, 1.0, total), top + torch.log(total)


def _packed_tensors(s):
    kv, dh = s["kv_heads"], s["dh"]
    at, there = _rows_of(s["cu"], s["longest"])
    q, k, v = (_grouped(s[x][at] * there[:, :, None], kv, dh) for x in "qkv")
    place = torch.arange(s["longest"], device="cuda")
    limit = (place if s["causal"] else torch.full_like(place, s["longest"])).expand(at.shape)
    p, lse = _probabilities(s, q, k, there, limit)
    return at, there, q, k, v, p, lse


def _packed_plain(s):
    seq, place, inside = _places(s["cu"], s["rows"])
    _, _, _, _, v, p, lse = _packed_tensors(s)
    out = _ungrouped(p @ v, s["longest"])[seq, place]
    lse = _ungrouped(lse, s["longest"])[seq, place]
    return (torch.where(inside[:, None], out, s["out"].float()).to(s["t"]),
            torch.where(inside[:, None], lse, s["lse"]))


def _packed_grad_plain(s):
    kv, dh, n = s["kv_heads"], s["dh"], s["longest"]
    seq, place, inside = _places(s["cu"], s["rows"])
    at, there, q, k, v, p, _ = _packed_tensors(s)
    do = _grouped(s["dout"][at] * there[:, :, None], kv, dh)
    dv = p.transpose(2, 3) @ do
    dp = do @ v.transpose(2, 3)
    ds = p * (dp - (p * dp).sum(3, keepdim=True)) * s["scale"]
    grads = _ungrouped(ds @ k, n), _ungrouped(ds.transpose(2, 3) @ q, n), _ungrouped(dv, n)
    return [torch.where(inside[:, None], x[seq, place], s[name].float()).to(s["t"])
            for x, name in zip(grads, ("dq", "dk", "dv"))]


def _quantise(x):
    """e4m3 bytes and E8M0 scale bytes of rows of 32-bit values: the scale is the least power of two, 2^-126 or more, that
    brings the largest value of the row within e4m3's 448; a row of zeros has scale 1."""
    top = x.abs().amax(-1)
    m, e = torch.frexp(top)
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-126)
    e = torch.where(top > 0, e, 0)
    return (torch.ldexp(x, -e[..., None])).to(torch.float8_e4m3fn).view(torch.uint8), (e + 127).to(torch.uint8)


def _dequantised(values, scale):
    return torch.ldexp(values.view(torch.float8_e4m3fn).float(), scale.int()[..., None] - 127)


def _new_slots(s):
    """(page, row in it) of each new token, and which rows are tokens."""
    seq, place, inside = _places(s["cu"], s["rows"])
    cu = s["cu"].long()
    position = s["kv_lens"].long()[seq] - (cu[1:] - cu[:-1])[seq] + place
    position = torch.where(inside, position, 0)
    return s["table"][seq, position // s["page"]].long(), position % s["page"], inside


def _write_plain(s):
    page, row, inside = _new_slots(s)
    at = (page * s["page"] + row)[inside]
    shape = (-1, s["kv_heads"], s["dh"])
    for x in "kv":
        new = s[x].reshape(shape)[inside]
        if s["cache"] == "e4m3":
            values, scale = _quantise(new.float())
            s[x + "_cache"].view(shape).index_copy_(0, at, values)
            s[x + "_scale"].view(shape[:2]).index_copy_(0, at, scale)
        else:
            s[x + "_cache"].view(shape).index_copy_(0, at, new)
    return _cache_out(s)


def _cache_out(s):
    if s["cache"] != "e4m3":
        return [s["k_cache"], s["v_cache"]]
    return [s["k_cache"].view(torch.float8_e4m3fn), s["v_cache"].view(torch.float8_e4m3fn),
            s["k_scale"].view(torch.float8_e8m0fnu), s["v_scale"].view(torch.float8_e8m0fnu)]


def _cached(s, x, page, row):
    """Rows of the cache in 32 bits, at page and row-in-page indices of any shape."""
    values = s[x + "_cache"][page, row]
    return _dequantised(values, s[x + "_scale"][page, row]) if s["cache"] == "e4m3" else values.float()


def _read_plain(s):
    page, row, _ = _new_slots(s)
    return [_cached(s, x, page, row).reshape(s["rows"], -1).to(s["t"]) for x in "kv"]


def _paged_plain(s):
    kv, dh = s["kv_heads"], s["dh"]
    at, there = _rows_of(s["cu"], s["longest_new"])
    q = _grouped(s["q"][at] * there[:, :, None], kv, dh)
    key = torch.arange(s["longest"], device="cuda")
    key_there = key < s["kv_lens"].long()[:, None]
    page = s["table"][:, key // s["page"]].long()
    k, v = (torch.where(key_there[:, :, None, None], _cached(s, x, page, (key % s["page"]).expand(page.shape)), 0.0)
            .transpose(1, 2) for x in "kv")
    new = (s["cu"][1:] - s["cu"][:-1]).long()
    limit = (s["kv_lens"].long() - new)[:, None] + torch.arange(s["longest_new"], device="cuda")
    p, _ = _probabilities(s, q, k, key_there, limit)
    seq, place, inside = _places(s["cu"], s["rows"])
    out = _ungrouped(p @ v, s["longest_new"])[seq, place]
    return torch.where(inside[:, None], out, s["out"].float()).to(s["t"])


# ---- the operators' own calls ------------------------------------------------------------------------------------

def _plan(s):
    """The descriptor a program keeps for its buffers, and the workspace beside it."""
    import ctypes

    from frame_hip import abi

    lib, code = abi.lib(), {"bf16": abi.BF16, "f16": abi.F16, "e4m3": abi.E4M3}
    if s["kind"] in ("fwd", "grad"):
        desc = abi.PackedAttention(dtype=code[s["dtype"]], causal=int(s["causal"]), tokens=s["rows"], batch=s["batch"],
                                   heads=s["heads"], kv_heads=s["kv_heads"], dh=s["dh"], q_stride=s["q"].stride(0),
                                   k_stride=s["k"].stride(0), v_stride=s["v"].stride(0), out_stride=s["out"].stride(0),
                                   scale=s["scale"])
        need = lib.fh_attention_packed_grad_workspace(ctypes.byref(desc)) if s["kind"] == "grad" else 0
    else:
        scales = [s[x + "_scale"].data_ptr() if s["cache"] == "e4m3" else None for x in "kv"]
        desc = abi.PagedCache(dtype=code[s["dtype"]], cache_dtype=code[s["cache"]], pages=s["pages"], page_size=s["page"],
                              kv_heads=s["kv_heads"], dh=s["dh"], k=s["k_cache"].data_ptr(), v=s["v_cache"].data_ptr(),
                              k_scale=scales[0], v_scale=scales[1], batch=s["batch"], block_table=s["table"].data_ptr(),
                              table_stride=s["table"].stride(0), kv_lens=s["kv_lens"].data_ptr())
        need = 0
        if s["kind"] == "paged":
            need = lib.fh_attention_paged_workspace(ctypes.byref(desc), s["rows"], s["heads"], s["longest_new"], s["longest"])
    assert need >= 0, abi.lib().fh_last_error()
    s["plan"] = abi, lib, desc, ctypes.byref(desc), torch.empty(max(need, 16), dtype=torch.uint8, device="cuda"), need
    return s["plan"]


def _run_own(s):
    abi, lib, desc, ref, ws, need = s.get("plan") or _plan(s)
    stream, kind = torch.cuda.current_stream().cuda_stream, s["kind"]
    if kind == "fwd":
        abi.check(lib.fh_attention_packed_fwd(ref, s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["cu"].data_ptr(),
                                              s["out"].data_ptr(), s["lse"].data_ptr(), stream))
        return [s["out"], s["lse"]]
    if kind == "grad":
        abi.check(lib.fh_attention_packed_grad(ref, s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["cu"].data_ptr(),
                                               s["out"].data_ptr(), s["lse"].data_ptr(), s["dout"].data_ptr(),
                                               s["dq"].data_ptr(), s["dk"].data_ptr(), s["dv"].data_ptr(), ws.data_ptr(), need,
                                               stream))
        return [s["dq"], s["dk"], s["dv"]]
    if kind == "write":
        abi.check(lib.fh_kv_cache_write(ref, s["k"].data_ptr(), s["k"].stride(0), s["v"].data_ptr(), s["v"].stride(0),
                                        s["rows"], s["cu"].data_ptr(), stream))
        return _cache_out(s)
    if kind == "read":
        abi.check(lib.fh_kv_cache_read(ref, s["k"].data_ptr(), s["k"].stride(0), s["v"].data_ptr(), s["v"].stride(0),
                                       s["rows"], s["cu"].data_ptr(), stream))
        return [s["k"], s["v"]]
    abi.check(lib.fh_attention_paged(ref, s["q"].data_ptr(), s["q"].stride(0), s["out"].data_ptr(), s["out"].stride(0),
                                     s["rows"], s["heads"], s["cu"].data_ptr(), s["scale"], s["longest_new"], s["longest"],
                                     ws.data_ptr(), need, stream))
    return [s["out"]]


def run(state):
    if own:
        return _run_own(state)
    kind = state["kind"]
    if kind == "fwd":
        return list(_packed_plain(state))
    if kind == "grad":
        return _packed_grad_plain(state)
    if kind == "write":
        return _write_plain(state)
    return _read_plain(state) if kind == "read" else [_paged_plain(state)]


# ---- from the definitions, in 64 bits ----------------------------------------------------------------------------

def _softmax64(scores):
    top = scores.max(-1, keepdim=True).values
    e = torch.exp(scores - top)
    total = e.sum(-1, keepdim=True)
    return e / total, (top + torch.log(total))[..., 0]


def _exact_packed(s):
    h, kv, dh = s["heads"], s["kv_heads"], s["dh"]
    at = [0] + list(_running(_ints(s["lens"])))
    heads = lambda x, b, j: x[at[b]:at[b + 1], j * dh:(j + 1) * dh].double()  # noqa: E731
    names = ("out", "lse") if s["kind"] == "fwd" else ("dq", "dk", "dv")
    got = {n: s[n].double().clone() for n in names}
    for b in range(s["batch"]):
        n = at[b + 1] - at[b]
        if n == 0:
            continue
        hidden = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1) if s["causal"] else None
        if s["kind"] == "grad":
            for x in names[1:]:
                got[x][at[b]:at[b + 1]] = 0
        for i in range(h):
            j = i * kv // h
            q, k, v = heads(s["q"], b, i), heads(s["k"], b, j), heads(s["v"], b, j)
            scores = torch.mm(q, k.t().contiguous()) / math.sqrt(dh)
            if hidden is not None:
                scores[hidden] = -math.inf
            p, lse = _softmax64(scores)
            rows, mine, shared = slice(at[b], at[b + 1]), slice(i * dh, (i + 1) * dh), slice(j * dh, (j + 1) * dh)
            if s["kind"] == "fwd":
                got["out"][rows, mine] = torch.mm(p, v)
                got["lse"][rows, i] = lse
                continue
            do = heads(s["dout"], b, i)
            dp = torch.mm(do, v.t().contiguous())
            got["dv"][rows, shared] += torch.mm(p.t().contiguous(), do)
            ds = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(dh)
            got["dq"][rows, mine] = torch.mm(ds, k)
            got["dk"][rows, shared] += torch.mm(ds.t().contiguous(), q)
    return [got[n] for n in names]


def _e4m3_values(b):
    """The values of e4m3 bytes: sign, 4 exponent bits (bias 7), 3 fraction bits."""
    b = b.long()
    e, f = (b >> 3) & 15, (b & 7).double()
    size = torch.where(e > 0, (8 + f) * torch.exp2((e - 10).double()), f * 2.0 ** -9)
    return torch.where(b >= 128, -size, size)


def _exact_rows(s, x, b, n):
    """Positions 0 .. n - 1 of sequence b: [n, kv_heads, dh]."""
    where = torch.arange(n, device="cuda")
    slot = s["table"][b].long()[where // s["page"]] * s["page"] + where % s["page"]
    raw = s[x + "_cache"].flatten(0, 1)[slot]
    if s["cache"] != "e4m3":
        return raw.double()
    return _e4m3_values(raw) * torch.exp2(s[x + "_scale"].flatten(0, 1)[slot].double() - 127)[..., None]


def _exact_written(s):
    """The cache after the write: the least power of two p with max|row| <= 448 p, and row / p on e4m3's grid, ties to even."""
    out = []
    caches = {}
    for x in "kv":
        cache = s[x + "_cache"].flatten(0, 1)
        caches[x] = (_e4m3_values(cache), torch.exp2(s[x + "_scale"].flatten(0, 1).double() - 127)) \
            if s["cache"] == "e4m3" else (cache.double(), None)
    at = [0] + list(_running(_ints(s["new"])))
    for b in range(s["batch"]):
        first = int(_ints(s["past"])[b])
        where = torch.arange(first, first + at[b + 1] - at[b], device="cuda")
        slot = s["table"][b].long()[where // s["page"]] * s["page"] + where % s["page"]
        for x in "kv":
            rows = s[x][at[b]:at[b + 1]].double().reshape(-1, s["kv_heads"], s["dh"])
            values, scales = caches[x]
            if scales is None:
                values[slot] = rows
                continue
            top = rows.abs().max(-1).values
            p = torch.exp2(torch.floor(torch.log2(top / 448)))
            p = torch.where(top > 448 * p, 2 * p, p)
            p = torch.where(top == 0, torch.ones_like(p), p)
            y = rows / p[..., None]
            step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
            values[slot], scales[slot] = torch.round(y / step) * step, p
    for i in range(2):
        for x in "kv":
            if caches[x][i] is not None:
                out.append(caches[x][i].reshape(s[x + "_cache"].shape[:4 - i]))
    return out


def _exact_paged(s):
    h, kv, dh = s["heads"], s["kv_heads"], s["dh"]
    out = s["out"].double().clone()
    at = [0] + list(_running(_ints(s["new"])))
    for b, past in enumerate(_ints(s["past"])):
        n = at[b + 1] - at[b]
        if n == 0:
            continue
        k, v = (_exact_rows(s, x, b, n + past) for x in "kv")
        hidden = torch.ones(n, n + past, dtype=torch.bool, device="cuda").triu(past + 1)
        q = s["q"][at[b]:at[b + 1]].double().reshape(n, h, dh)
        for j in range(kv):
            mine = slice(j * h // kv, (j + 1) * h // kv)
            kj, vj = k[:, j].contiguous(), v[:, j].contiguous()
            scores = torch.mm(q[:, mine].reshape(-1, dh), kj.t().contiguous()).reshape(n, -1, n + past) / math.sqrt(dh)
            p, _ = _softmax64(scores.masked_fill(hidden[:, None], -math.inf))
            got = torch.mm(p.reshape(-1, n + past), vj)
            out[at[b]:at[b + 1]].reshape(n, h, dh)[:, mine] = got.reshape(n, -1, dh)
    return [out]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("fwd", "grad"):
        return _exact_packed(s)
    if case["kind"] == "write":
        return _exact_written(s)
    if case["kind"] == "paged":
        return _exact_paged(s)
    rows = [[_exact_rows(s, x, b, n).flatten(1) for b, n in enumerate(_ints(s["lens"]))] for x in "kv"]
    return [torch.cat(r) for r in rows]
