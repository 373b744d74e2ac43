"""The token head's operators (pst_amd.head): what is measured, their plain forms and their definitions in 64 bits.

A token head is a table `weight` [V, d] with one row per token id: the codes of a codebook (432, 1728, 4096 or
64000 of them) and, usually, a few marks (begin, end, padding). `hidden` [N, d] is what a sequence model over
token ids holds at N positions.

  loss    loss[n] = lse[n] - logit[n, target[n]], lse[n] = log sum_v exp(logit[n, v]), logit = hidden weight^T
  grad    the gradients of sum_n grad_loss[n] loss[n] for hidden and weight
  scores  logits in 8-bit integers: hidden is rounded to 8 bits with a scale for each row, weight was before
"""
import math
import os
import sys

import torch

own = False

IGNORE = -100
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
LARGEST = 8192 * 64003 * 1024


def listed():
    return [
        # the loss of one protein of the fewest residues that the tokenizer takes, a narrow model: latency
        dict(name="loss-one-protein", op="loss", rows=50, vocab=4096, width=128, type="bf16", pad=0),
        # scoring eight proteins of 512 residues under the 4096 codes and three marks
        dict(name="loss-batch", op="loss", rows=4096, vocab=4099, width=512, type="bf16", pad=0),
        # a training step's loss over the large codebook
        dict(name="loss-64k", op="loss", rows=8192, vocab=64003, width=1024, type="bf16", pad=0),
        # a model kept in 32 bits; its hidden states are a slice of a wider buffer, and the width is odd
        dict(name="loss-f32-odd", op="loss", rows=1023, vocab=4099, width=333, type="f32", pad=7),
        # gradients of one short protein
        dict(name="grad-one-protein", op="grad", rows=50, vocab=4096, width=128, type="f16", pad=0),
        # a small model's training step
        dict(name="grad-batch", op="grad", rows=4096, vocab=4099, width=512, type="bf16", pad=0),
        # a training step over the large codebook
        dict(name="grad-64k", op="grad", rows=8192, vocab=64003, width=1024, type="bf16", pad=0),
        # a model kept in 32 bits
        dict(name="grad-f32", op="grad", rows=1000, vocab=4096, width=512, type="f32", pad=0),
        # answering: one token of one sequence
        dict(name="scores-one", op="scores", rows=1, vocab=4096, width=512, type="bf16", out="f32", pad=0),
        # answering: one token of each of 16 sequences over the large codebook
        dict(name="scores-16", op="scores", rows=16, vocab=64003, width=1024, type="bf16", out="bf16", pad=0),
        # scoring whole sequences of a model kept in 32 bits, odd sizes
        dict(name="scores-odd", op="scores", rows=2047, vocab=4099, width=700, type="f32", out="f32", pad=5),
        # scoring many positions over the large codebook
        dict(name="scores-64k", op="scores", rows=8192, vocab=64003, width=1024, type="f16", out="bf16", pad=0),
    ]


def draw(rng):
    def over(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["loss", "grad", "scores"])
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    vocab = rng.choice([432, 1728, 4096, 64000]) + rng.choice([0, 0, 1, 3, 64]) if rng.random() < 0.7 else over(2, 64064)
    width = rng.choice([64, 128, 256, 384, 512, 768, 1024, 1536, 2048]) if rng.random() < 0.6 else over(16, 2048)
    rows = over(1, 8192)
    limit = LARGEST // (6 if kind == "f32" else 1)  # 32-bit products cost a multiple of 16-bit ones
    rows = max(1, min(rows, limit // (vocab * width)))
    case = dict(op=op, rows=rows, vocab=vocab, width=width, type=kind, pad=rng.choice([0, 0, 0, 1, 8, 24]))
    if op == "scores":
        case["out"] = rng.choice(["f32", "bf16", "f16"])
    return case


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, vocab, width, kind = case["rows"], case["vocab"], case["width"], TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    # rows of the table of about unit length, normalised hidden states that point towards their target's row: losses
    # between those of an untrained and of a trained model
    weight = normal(vocab, width) * (1.5 / math.sqrt(width))
    targets = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    hidden = normal(rows, width) + 2.0 * torch.rand(rows, 1, generator=g, device="cuda") * weight[targets]
    held = torch.zeros(rows, width + case["pad"], device="cuda", dtype=kind)
    hidden = held[:, :width].copy_(hidden)
    state = dict(case=case, hidden=hidden)
    if case["op"] == "scores":
        scale = weight.abs().amax(1) / 127.0
        state["weight"] = torch.round(weight / scale[:, None]).to(torch.int8)
        state["scale"] = scale
        return state
    weight = weight.to(kind)
    # an eighth of the positions carry no loss: the padding behind shorter proteins
    targets[torch.rand(rows, generator=g, device="cuda") < 0.125] = IGNORE
    state["weight"], state["targets"] = weight, targets
    if case["op"] == "grad":
        state["lse"] = torch.logsumexp(hidden.float() @ weight.float().T, 1)  # of the forward pass
        # a mean over the positions, each with a weight of its own; f16 is trained with a scaled loss
        scaled = 2048.0 if case["type"] == "f16" else 1.0
        state["grad_loss"] = (0.5 + torch.rand(rows, generator=g, device="cuda")) * (scaled / rows)
    return state


def run(state):
    op, hidden, weight = state["case"]["op"], state["hidden"], state["weight"]
    if own:
        head = framework()
        if op == "loss":
            return head.token_loss(hidden, weight, state["targets"], ignore_index=IGNORE)
        if op == "grad":
            return head.token_loss_grad(hidden, weight, state["targets"], state["lse"], state["grad_loss"], ignore_index=IGNORE)
        return head.token_scores_int8(hidden, weight, state["scale"], out_dtype=TYPES[state["case"]["out"]])
    if op == "loss":
        return plain_loss(hidden, weight, state["targets"])
    if op == "grad":
        return plain_grad(hidden, weight, state["targets"], state["lse"], state["grad_loss"])
    return plain_scores(hidden, weight, state["scale"], TYPES[state["case"]["out"]])


def framework():
    at = os.path.join(os.getcwd(), "protein-structure-tokenizer_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from pst_amd import head
    return head


def plain_loss(hidden, weight, targets):
    logits = hidden.float() @ weight.float().T
    top = logits.amax(1)
    lse = top + (logits - top[:, None]).exp().sum(1).log()
    valid = targets != IGNORE
    at = logits.gather(1, torch.where(valid, targets, 0)[:, None])[:, 0]
    return torch.where(valid, lse - at, 0.0), lse


def plain_grad(hidden, weight, targets, lse, grad_loss):
    h, w = hidden.float(), weight.float()
    valid = targets != IGNORE
    d = (h @ w.T - lse[:, None]).exp()
    d.scatter_add_(1, torch.where(valid, targets, 0)[:, None], torch.full_like(lse, -1.0)[:, None])
    d *= torch.where(valid, grad_loss, 0.0)[:, None]
    return (d @ w).to(hidden.dtype), (d.T @ h).to(weight.dtype)


def plain_scores(hidden, weight, scale, out):
    h = hidden.float()
    s = h.abs().amax(1) / 127.0
    q = torch.round(h / torch.where(s > 0, s, 1.0)[:, None])
    return (q @ weight.float().T * s[:, None] * scale).to(out)


def work(case):
    n, v, d, e = case["rows"], case["vocab"], case["width"], BYTES[case["type"]]
    if case["op"] == "loss":
        return {"bytes": e * (n + v) * d + 16 * n, "flops": 2 * n * v * d}
    if case["op"] == "grad":
        return {"bytes": 2 * e * (n + v) * d + 16 * n, "flops": 6 * n * v * d}
    return {"bytes": e * n * d + v * (d + 4) + BYTES[case["out"]] * n * v, "flops": 2 * n * v * d}


def exact(case, seed):
    """From the definitions, one row of hidden at a time in the formulas, all in 64 bits."""
    state = prepare(case, seed)
    x, w = state["hidden"].double(), state["weight"].double()
    if case["op"] == "scores":
        # the rounding to 8 bits is the operator's, in 32 bits: its integers are exact from there on
        largest = state["hidden"].float().abs().max(dim=1).values
        step = torch.div(largest, 127.0)
        codes = torch.nan_to_num(torch.div(state["hidden"].float(), step.unsqueeze(1))).round().double()
        return torch.mm(codes, w.t()).mul_(step.double().unsqueeze(1)).mul_(state["scale"].double().unsqueeze(0))
    logits = torch.mm(x, w.t())
    rows = torch.nonzero(state["targets"] != IGNORE).flatten()
    at = state["targets"][rows]
    if case["op"] == "loss":
        lse = torch.logsumexp(logits, dim=1)
        loss = torch.zeros_like(lse)
        loss[rows] = lse[rows] - logits[rows, at]
        return loss, lse
    # d loss / d logit = softmax - indicator; lse is an input here, as it is of the operator
    slope = torch.exp(logits[rows].sub_(state["lse"].double()[rows].unsqueeze(1)))
    del logits
    slope[torch.arange(rows.numel(), device=rows.device), at] -= 1
    slope *= state["grad_loss"].double()[rows].unsqueeze(1)
    dx = torch.zeros_like(x)
    dx[rows] = slope.mm(w)
    return dx, slope.t().mm(x[rows])
