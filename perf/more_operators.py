"""The two ends of a language model, as measurable cases: token embedding and the loss over the vocabulary, each with its gradient.

Each case is one call of one operator on buffers that a program keeps on the GPU:

  embed       a row of the table for every token, times a scale; tokens outside the vocabulary get zeros
  embed_grad  the table's gradient: the sum of the tokens' rows per id, on zeros or on top of another gradient of the same table
  loss        softmax cross entropy of x w^T against integer targets, per row and as a mean; rows without a target do not count
  loss_grad   its gradients with respect to x and w, from the forward's log-sum-exp

`own` false: elementary torch operations in 32 bits, rounded once at the end. `own` true: the kernel library's entry points.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if os.path.join(REPO, "frame-public_amd") not in sys.path:
    sys.path.insert(0, os.path.join(REPO, "frame-public_amd"))

TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---- the cases --------------------------------------------------------------------------------------------------

def listed():
    return [
        # a decoding step's 64 sequences: one row each, launch and latency
        dict(name="embed_step", kind="embed", dtype="bf16", tokens=64, vocab=32768, dim=1024, scale=1.0, outside=0.0),
        # a long prompt of a wide model whose table is multiplied by sqrt(dim), some rows padding
        dict(name="embed_prompt", kind="embed", dtype="bf16", tokens=8192, vocab=131072, dim=4096, scale=64.0, outside=0.05),
        # a small odd model in 32 bits, rows that no 16-byte vector divides
        dict(name="grad_odd", kind="embed_grad", dtype="f32", tokens=301, vocab=5003, dim=333, scale=1.0, outside=0.0, add=False),
        # the transformer block's batch (8 x 512 tokens of 1,024), on top of the tied output projection's gradient
        dict(name="grad_tied", kind="embed_grad", dtype="bf16", tokens=4096, vocab=32768, dim=1024, scale=1.0, outside=0.0,
             add=True),
        # a long-context training step of a wide model: the whole table's gradient is written
        dict(name="grad_long", kind="embed_grad", dtype="bf16", tokens=32768, vocab=131072, dim=4096, scale=1.0, outside=0.1,
             add=False),
        # the score of a single token, as a serving step has it: the table's bytes
        dict(name="loss_one", kind="loss", dtype="bf16", tokens=1, vocab=131072, dim=4096, outside=0.0),
        # an evaluation of a few short answers, odd sizes, prompts without targets
        dict(name="loss_odd", kind="loss", dtype="f16", tokens=333, vocab=50261, dim=1000, outside=0.4),
        # the transformer block's batch
        dict(name="loss_block", kind="loss", dtype="bf16", tokens=4096, vocab=32768, dim=1024, outside=0.0),
        # a wide model's training batch with padding
        dict(name="loss_long", kind="loss", dtype="bf16", tokens=8192, vocab=131072, dim=4096, outside=0.1),
        # a small fine-tuning step, odd sizes, prompts without targets
        dict(name="loss_grad_odd", kind="loss_grad", dtype="f16", tokens=333, vocab=5003, dim=1000, outside=0.4),
        # the transformer block's batch, backward
        dict(name="loss_grad_block", kind="loss_grad", dtype="bf16", tokens=4096, vocab=32768, dim=1024, outside=0.0),
        # a wide model's training batch, backward
        dict(name="loss_grad_long", kind="loss_grad", dtype="bf16", tokens=4096, vocab=131072, dim=4096, outside=0.1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One case of the ranges above: tokens from one to a long batch, vocabularies of any size, widths over their logarithm."""
    kind = rng.choice(["embed", "embed_grad", "embed_grad", "loss", "loss", "loss_grad", "loss_grad"])
    outside = rng.choice([0.0, 0.0, 0.1, 0.5])
    vocab = _log_int(rng, 500, 131072)
    if kind in ("embed", "embed_grad"):
        case = dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), tokens=_log_int(rng, 1, 32768), vocab=vocab,
                    dim=rng.choice([1, 1, 8, 8, 64]) * _log_int(rng, 16, 64) if rng.random() < 0.7 else _log_int(rng, 16, 2048),
                    scale=rng.choice([1.0, 1.0, 22.627417, 0.5]), outside=outside)
        if kind == "embed_grad":
            case["add"] = rng.random() < 0.4
        return case
    while True:
        case = dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "f16"]), tokens=_log_int(rng, 1, 8192), vocab=vocab,
                    dim=8 * _log_int(rng, 8, 512), outside=outside)
        if case["tokens"] * case["vocab"] * case["dim"] <= 2 ** 40:
            return case


# ---- work -------------------------------------------------------------------------------------------------------

def _counted(case):
    """Tokens with an id (or a target) inside the vocabulary; at least one."""
    return max(1, case["tokens"] - int(round(case["outside"] * case["tokens"])))


def _distinct(case):
    """How many different ids the counted tokens are expected to have (see _ids)."""
    v = np.arange(1, case["vocab"] + 1, dtype=np.float64)
    p = np.log1p(1.0 / v) / math.log(case["vocab"] + 1)
    return float(-np.expm1(_counted(case) * np.log1p(-p)).sum())


def work(case):
    n, m, v, d = case["tokens"], _counted(case), case["vocab"], case["dim"]
    e = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "embed":  # the rows that are named, once; a row out per token
        return {"bytes": int(4 * n + e * d * (_distinct(case) + n)), "flops": 0}
    if case["kind"] == "embed_grad":  # counted rows and the other gradient in; the table's gradient out
        return {"bytes": 4 * n + e * d * (m + (2 if case["add"] else 1) * v), "flops": m * d}
    if case["kind"] == "loss":  # x, w, targets in; row losses and log-sum-exps out
        return {"bytes": e * d * (m + v) + 12 * n, "flops": 2 * m * v * d}
    # x, w, targets, log-sum-exps in; dx and dw out
    return {"bytes": e * d * (m + v + n + v) + 8 * n, "flops": 6 * m * v * d}


# ---- inputs -----------------------------------------------------------------------------------------------------

def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _ids(case, g):
    """Ids with the frequencies of words in a text (proportional to 1 / rank, nearly), -1 for tokens outside the vocabulary."""
    n, v = case["tokens"], case["vocab"]
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    ids = (torch.exp(u * math.log(v + 1)).long() - 1).clamp(0, v - 1)
    out = torch.randperm(n, generator=g, device="cuda")[:n - _counted(case)]
    ids[out] = -1
    return ids.to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    n, v, d, t = s["tokens"], s["vocab"], s["dim"], TORCH[s["dtype"]]
    s["t"] = t
    s["ids"] = _ids(case, g)
    if s["kind"] == "embed":
        s["table"] = _randn(g, v, d).to(t)
        s["out"] = torch.empty(n, d, dtype=t, device="cuda")
    elif s["kind"] == "embed_grad":
        s["dout"] = _randn(g, n, d).to(t)
        s["base"] = _randn(g, v, d).to(t) if s["add"] else None  # the gradient from the table's other use
        s["dtable"] = torch.empty(v, d, dtype=t, device="cuda")
    else:
        # logits of deviation 1.5; a model that has learned something: most targets' logits are raised, by 2 to 14
        w = _randn(g, v, d).mul_(1.5 / math.sqrt(d))
        x = _randn(g, n, d)
        mine = w[s["ids"].long().clamp(min=0)]
        x += mine * ((2 + 12 * torch.rand(n, 1, generator=g, device="cuda")) / mine.square().sum(1, keepdim=True))
        s["x"], s["w"] = x.to(t), w.to(t)
        del x, w, mine
        s["lse"] = torch.empty(n, device="cuda")
        if s["kind"] == "loss":
            s["loss"] = torch.empty((), device="cuda")
            s["row_loss"] = torch.empty(n, device="cuda")
        else:
            s["dloss"] = torch.full((), 1024.0 if s["dtype"] == "f16" else 1.0, device="cuda")  # f16 steps scale their loss
            s["lse"].copy_(_loss_plain(s)[2])
            s["dx"] = torch.empty(n, d, dtype=t, device="cuda")
            s["dw"] = torch.empty(v, d, dtype=t, device="cuda")
    return s


# ---- the operators in their plain form ---------------------------------------------------------------------------

def _embed_plain(s):
    ids = s["ids"].long()
    there = (ids >= 0) & (ids < s["vocab"])
    rows = s["table"][torch.where(there, ids, 0)].float() * s["scale"]
    return torch.where(there[:, None], rows, 0.0).to(s["t"])


def _embed_grad_plain(s):
    ids = s["ids"].long()
    there = (ids >= 0) & (ids < s["vocab"])
    total = torch.zeros(s["vocab"], s["dim"], device="cuda")
    total.index_add_(0, torch.where(there, ids, 0), s["dout"].float() * (there * s["scale"])[:, None])
    if not s["add"]:
        return total.to(s["t"])
    return (s["base"].float() + total).to(s["t"])


def _logits(s):
    ids = s["ids"].long()
    there = (ids >= 0) & (ids < s["vocab"])
    return torch.mm(s["x"].float(), s["w"].float().t()), torch.where(there, ids, 0), there


def _loss_plain(s):
    z, target, there = _logits(s)
    top = z.amax(1, keepdim=True)
    lse = (top + torch.log(torch.exp(z - top).sum(1, keepdim=True)))[:, 0]
    row = lse - z.gather(1, target[:, None])[:, 0]
    row, lse = torch.where(there, row, 0.0), torch.where(there, lse, 0.0)
    return [row.double().sum().float() / there.sum(), row, lse]


def _loss_grad_plain(s):
    z, target, there = _logits(s)
    p = torch.exp(z - s["lse"][:, None])
    p[torch.arange(s["tokens"], device="cuda"), target] -= 1.0
    p = torch.where(there[:, None], p, 0.0)
    f = s["dloss"] / there.sum()
    return [(torch.mm(p, s["w"].float()) * f).to(s["t"]), (torch.mm(p.t(), s["x"].float()) * f).to(s["t"])]


# ---- the operators' own calls ------------------------------------------------------------------------------------

def _plan(s):
    """The descriptor a program keeps for its buffers, and the workspace beside it."""
    import ctypes

    from frame_hip import abi

    lib, code = abi.lib(), {"bf16": abi.BF16, "f16": abi.F16, "f32": abi.F32}
    need = 0
    if s["kind"] in ("embed", "embed_grad"):
        desc = abi.TokenEmbedding(dtype=code[s["dtype"]], tokens=s["tokens"], vocab=s["vocab"], dim=s["dim"],
                                  row_stride=s["dim"], scale=s["scale"])
        if s["kind"] == "embed_grad":
            need = lib.fh_embedding_grad_workspace(ctypes.byref(desc))
    else:
        desc = abi.VocabLoss(dtype=code[s["dtype"]], loss_dtype=abi.F32, mean=1, tokens=s["tokens"], vocab=s["vocab"],
                             dim=s["dim"], x_stride=s["dim"], w_stride=s["dim"])
        query = lib.fh_vocab_loss_workspace if s["kind"] == "loss" else lib.fh_vocab_loss_grad_workspace
        need = query(ctypes.byref(desc))
    assert need >= 0, lib.fh_last_error()
    s["plan"] = abi, lib, desc, ctypes.byref(desc), torch.empty(max(need, 16), dtype=torch.uint8, device="cuda"), need
    return s["plan"]


def _run_own(s):
    abi, lib, desc, ref, ws, need = s.get("plan") or _plan(s)
    stream, kind = torch.cuda.current_stream().cuda_stream, s["kind"]
    if kind == "embed":
        abi.check(lib.fh_embedding_fwd(ref, s["table"].data_ptr(), s["ids"].data_ptr(), s["out"].data_ptr(), stream))
        return [s["out"]]
    if kind == "embed_grad":
        abi.check(lib.fh_embedding_grad(ref, s["dout"].data_ptr(), s["ids"].data_ptr(),
                                        s["base"].data_ptr() if s["add"] else None, s["dtable"].data_ptr(), ws.data_ptr(), need,
                                        stream))
        return [s["dtable"]]
    if kind == "loss":
        abi.check(lib.fh_vocab_loss_fwd(ref, s["x"].data_ptr(), s["w"].data_ptr(), s["ids"].data_ptr(), s["loss"].data_ptr(),
                                        s["row_loss"].data_ptr(), s["lse"].data_ptr(), ws.data_ptr(), need, stream))
        return [s["loss"], s["row_loss"], s["lse"]]
    abi.check(lib.fh_vocab_loss_grad(ref, s["x"].data_ptr(), s["w"].data_ptr(), s["ids"].data_ptr(), s["lse"].data_ptr(),
                                     s["dloss"].data_ptr(), s["dx"].data_ptr(), s["dw"].data_ptr(), ws.data_ptr(), need, stream))
    return [s["dx"], s["dw"]]


def run(state):
    if own:
        return _run_own(state)
    kind = state["kind"]
    if kind == "embed":
        return [_embed_plain(state)]
    if kind == "embed_grad":
        return [_embed_grad_plain(state)]
    return _loss_plain(state) if kind == "loss" else _loss_grad_plain(state)


# ---- from the definitions, in 64 bits ----------------------------------------------------------------------------

def _exact_embed(s):
    out = torch.zeros(s["tokens"], s["dim"], dtype=torch.float64, device="cuda")
    inside = s["ids"] >= 0
    out[inside] = s["table"][s["ids"][inside].long()].double() * s["scale"]
    return [out]


def _exact_embed_grad(s):
    """Tokens sorted by id; each id's rows are the difference of two running sums, in pieces of the columns."""
    out = s["base"].double() if s["add"] else torch.zeros(s["vocab"], s["dim"], dtype=torch.float64, device="cuda")
    ids, order = torch.sort(s["ids"][s["ids"] >= 0].long(), stable=True)
    order = torch.nonzero(s["ids"] >= 0)[:, 0][order]
    names, counts = torch.unique_consecutive(ids, return_counts=True)
    ends = counts.cumsum(0)
    for at in range(0, s["dim"], 512):
        run_ = s["dout"][order, at:at + 512].double().cumsum(0)
        run_ = torch.cat([torch.zeros_like(run_[:1]), run_])
        out[names, at:at + 512] += (run_[ends] - run_[ends - counts]) * s["scale"]
    return [out]


def _exact_loss(s, grad):
    n, step = s["tokens"], 1024
    w = s["w"].double()
    wt = w.t().contiguous()
    counted = torch.nonzero(s["ids"] >= 0)[:, 0]
    lse, row = (torch.zeros(n, dtype=torch.float64, device="cuda") for _ in "ab")
    dx = torch.zeros(n, s["dim"], dtype=torch.float64, device="cuda") if grad else None
    dw = torch.zeros_like(w) if grad else None
    for at in range(0, counted.numel(), step):
        mine = counted[at:at + step]
        x, target = s["x"][mine].double(), s["ids"][mine].long()
        z = torch.mm(x, wt)
        lse[mine] = torch.logsumexp(z, 1)
        row[mine] = lse[mine] - z.gather(1, target[:, None])[:, 0]
        if grad:
            z.sub_(lse[mine][:, None]).exp_()
            z.scatter_add_(1, target[:, None], torch.full_like(target[:, None], -1.0, dtype=torch.float64))
            z.mul_(s["dloss"].double() / counted.numel())
            dx[mine] = torch.mm(z, w)
            dw += torch.mm(z.t().contiguous(), x)
    return [dx, dw] if grad else [row.sum() / counted.numel(), row, lse]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "embed":
        return _exact_embed(s)
    if case["kind"] == "embed_grad":
        return _exact_embed_grad(s)
    return _exact_loss(s, case["kind"] == "loss_grad")
