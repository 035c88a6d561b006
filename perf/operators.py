"""What the operators at the two ends of a language model are measured on: the embedding of its tokens and the losses of its head.

  embed   ``scale * weight[ids] + position_weight[positions]``, with the gradients of both tables
  ce      softmax cross entropy of ``x @ weight.T`` over the vocabulary, with the gradients of ``x`` and ``weight``
  kd      distillation from a teacher's top logits over the same product, with the same gradients

All three read a table of [vocabulary, width].  ``own`` selects the framework's operators; otherwise the same results come
from elementary torch operations in 32 bits, rounded once.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32, "fp16": torch.float16}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
IGNORED = -100


def listed():
    return [
        # the lookup of one generated token: latency only
        {"name": "embed_token", "op": "embed", "n": 1, "v": 50257, "d": 1024, "dtype": "bf16", "grad": False, "pos": 1024, "scale": 1.0, "pad": False},
        # the first stage of a GPT-2 medium training step: 8 sequences of 1024 tokens with learned positions
        {"name": "embed_step", "op": "embed", "n": 8192, "v": 50257, "d": 1024, "dtype": "bf16", "grad": True, "pos": 1024, "scale": 1.0, "pad": False},
        # odd numbers of tokens and columns, fp32 table, scaled rows, no positions, a padding token
        {"name": "embed_ragged", "op": "embed", "n": 5003, "v": 30011, "d": 500, "dtype": "fp32", "grad": True, "pos": 0, "scale": 22.36, "pad": True},
        # a large batch: 128 sequences of 1024 tokens
        {"name": "embed_long", "op": "embed", "n": 131072, "v": 50257, "d": 1024, "dtype": "bf16", "grad": True, "pos": 1024, "scale": 1.0, "pad": False},
        # scoring a short text: one loss per token, no gradients
        {"name": "ce_score", "op": "ce", "n": 77, "v": 50257, "d": 1024, "grad": False, "reduction": "none", "ignored": 0.0},
        # GPT-2 tiny: 8 sequences of 128 tokens, 512 tokens in the vocabulary
        {"name": "ce_tiny", "op": "ce", "n": 1024, "v": 512, "d": 256, "grad": True, "reduction": "mean", "ignored": 0.0},
        # a ragged batch with padding: an odd number of rows, a tenth of them ignored, one gradient per row
        {"name": "ce_ragged", "op": "ce", "n": 2003, "v": 50257, "d": 768, "grad": True, "reduction": "none", "ignored": 0.1},
        # the head of a GPT-2 medium training step
        {"name": "ce_step", "op": "ce", "n": 8192, "v": 50257, "d": 1024, "grad": True, "reduction": "mean", "ignored": 0.0},
        # the same for four such batches at once
        {"name": "ce_long", "op": "ce", "n": 32768, "v": 50257, "d": 1024, "grad": True, "reduction": "mean", "ignored": 0.02},
        # a validation pass of a distilled model: losses only, short lists
        {"name": "kd_score", "op": "kd", "n": 509, "v": 50257, "d": 768, "k": 8, "temp": 1.0, "grad": False, "reduction": "none", "masked": 0.0},
        # a ragged batch: lists of different lengths, some rows without any entry
        {"name": "kd_ragged", "op": "kd", "n": 1777, "v": 30011, "d": 640, "k": 17, "temp": 1.5, "grad": True, "reduction": "sum", "masked": 0.3},
        # a distillation step of a GPT-2 medium student
        {"name": "kd_step", "op": "kd", "n": 8192, "v": 50257, "d": 1024, "k": 32, "temp": 2.0, "grad": True, "reduction": "mean", "masked": 0.05},
    ]


def _log(rng, low, high):
    """Log-uniform whole number of [low, high]."""
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    op = rng.choice(["embed", "ce", "ce", "kd"])
    v = _log(rng, 500, 50257)
    grad = rng.random() < 0.75
    if op == "embed":
        return {"op": op, "n": _log(rng, 1, 131072), "v": v, "d": rng.choice([1, 2, 4, 8]) * rng.randint(32, 128), "dtype": rng.choice(["bf16", "bf16", "fp32", "fp16"]),
                "grad": grad, "pos": rng.choice([0, 128, 1000, 1024]), "scale": rng.choice([1.0, 16.0, 22.36]), "pad": rng.random() < 0.3}
    case = {"op": op, "n": _log(rng, 1, 16384), "v": v, "d": 8 * _log(rng, 8, 160), "grad": grad, "reduction": rng.choice(["mean", "sum", "none"])}
    if op == "ce":
        case["ignored"] = rng.choice([0.0, 0.1, 0.5])
    else:
        case.update(k=_log(rng, 1, 64), temp=rng.choice([1.0, 2.0, 3.5]), masked=rng.choice([0.0, 0.3]))
    return case


def _tokens(g, n, v):
    """Token ids as texts have them: a few very often, many hardly ever."""
    u = torch.rand(n, generator=g, device="cuda")
    rank = (torch.exp(u * math.log(v + 1.0)) - 1.0).long().clamp_(0, v - 1)
    return (rank * 7919 + 13) % v


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, v, d = case["n"], case["v"], case["d"]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * std

    s = dict(case)
    if case["op"] == "embed":
        dt = DTYPES[case["dtype"]]
        s["weight"] = normal(v, d, std=0.02).to(dt).requires_grad_(case["grad"])
        s["ids"] = _tokens(g, n, v)
        s["padding"] = int(s["ids"][0]) if case["pad"] else None
        if case["pos"]:
            s["pweight"] = normal(case["pos"], d, std=0.02).to(dt).requires_grad_(case["grad"])
            s["positions"] = torch.arange(n, device="cuda") % case["pos"]
        if case["grad"]:
            s["gout"] = normal(n, d, std=1e-2).to(dt)
        return s
    # rows as a layer norm leaves them, a head that has learned something: the targets' logits stand out by a few units
    w = normal(v, d, std=0.02)
    t = _tokens(g, n, v)
    x = normal(n, d) + w[t] * (torch.rand(n, 1, generator=g, device="cuda") * 12.0 / (0.02 * 0.02 * d))
    s["weight"], s["x"] = w.to(torch.bfloat16).requires_grad_(case["grad"]), x.to(torch.bfloat16).requires_grad_(case["grad"])
    if case["op"] == "ce":
        drop = torch.rand(n, generator=g, device="cuda") < case["ignored"]
        s["targets"] = torch.where(drop, IGNORED, t)
    else:
        k = case["k"]
        step = torch.randint(1, max(2, v // k), (n, 1), generator=g, device="cuda")
        tokens = (t[:, None] + step * torch.arange(k, device="cuda")) % v        # a row's tokens are all different
        s["tlogits"] = normal(n, k, std=1.5).sort(dim=1, descending=True).values + 8.0
        length = torch.where(torch.rand(n, 1, generator=g, device="cuda") < case["masked"], torch.randint(0, k + 1, (n, 1), generator=g, device="cuda"), k)
        s["ttokens"] = torch.where(torch.arange(k, device="cuda") < length, tokens, -1)
    if case["grad"] and case["reduction"] == "none":
        s["gout"] = torch.rand(n, generator=g, device="cuda") / n
    return s


def run(s):
    if own:
        return {"embed": _own_embed, "ce": _own_ce, "kd": _own_kd}[s["op"]](s)
    with torch.no_grad():
        return {"embed": _plain_embed, "ce": _plain_ce, "kd": _plain_kd}[s["op"]](s)


# ---------------------------------------------------------------- the framework's operators
def _own_embed(s):
    from dfccl_b200.ops.embedding import embedding
    out = embedding(s["ids"], s["weight"], scale=s["scale"], padding_idx=s["padding"], positions=s.get("positions"), position_weight=s.get("pweight"))
    if not s["grad"]:
        return {"out": out}
    tables = [s["weight"]] + ([s["pweight"]] if s["pos"] else [])
    return {"out": out.detach(), "grads": torch.autograd.grad(out, tables, s["gout"])}


def _own_loss(s, loss):
    if not s["grad"]:
        return {"loss": loss}
    dx, dw = torch.autograd.grad(loss, [s["x"], s["weight"]], s.get("gout"))
    return {"loss": loss.detach(), "dx": dx, "dw": dw}


def _own_ce(s):
    from dfccl_b200.ops.loss import linear_cross_entropy
    return _own_loss(s, linear_cross_entropy(s["x"], s["weight"], s["targets"], ignore_index=IGNORED, reduction=s["reduction"]))


def _own_kd(s):
    from dfccl_b200.ops.loss import linear_distillation
    return _own_loss(s, linear_distillation(s["x"], s["weight"], s["tlogits"], s["ttokens"], temperature=s["temp"], reduction=s["reduction"]))


# ---------------------------------------------------------------- plain forms, 32 bits
def _plain_embed(s):
    w, ids = s["weight"], s["ids"]
    y = w[ids].float() * s["scale"]
    if s["pos"]:
        y = y + s["pweight"][s["positions"]].float()
    out = y.to(w.dtype)
    if not s["grad"]:
        return {"out": out}
    g = s["gout"].float()
    gw = torch.zeros(w.shape, dtype=torch.float32, device="cuda")
    gs = g * s["scale"]
    if s["padding"] is not None:
        gs = gs * (ids != s["padding"])[:, None]
    gw.index_add_(0, ids, gs)
    grads = [gw.to(w.dtype)]
    if s["pos"]:
        gp = torch.zeros(s["pweight"].shape, dtype=torch.float32, device="cuda")
        gp.index_add_(0, s["positions"], g)
        grads.append(gp.to(w.dtype))
    return {"out": out, "grads": tuple(grads)}


def _reduced(s, loss, valid):
    """The loss as asked for, and what every row's loss counts in it."""
    if s["reduction"] == "none":
        return loss, s.get("gout")
    if s["reduction"] == "sum":
        return loss.sum(), valid.float()
    count = valid.sum().float()
    share = torch.where(count > 0, 1.0 / count, torch.zeros_like(count))
    return loss.sum() * share, valid.float() * share


def _plain_grads(s, p, x, w, loss):
    """Gradients of x and w from p, that of the logits."""
    return {"loss": loss, "dx": (p @ w).to(torch.bfloat16), "dw": (p.t() @ x).to(torch.bfloat16)}


def _plain_ce(s):
    x, w, t = s["x"].float(), s["weight"].float(), s["targets"]
    valid = t != IGNORED
    col = torch.where(valid, t, 0)
    z = x @ w.t()
    top = z.max(dim=1, keepdim=True).values
    e = torch.exp(z - top)
    total = e.sum(dim=1, keepdim=True)
    loss = (torch.log(total) + top - z.gather(1, col[:, None]))[:, 0]
    loss, share = _reduced(s, torch.where(valid, loss, 0.0), valid)
    if not s["grad"]:
        return {"loss": loss}
    p = e.div_(total)
    p[torch.arange(t.numel(), device="cuda"), col] -= 1.0
    p.mul_((share * valid)[:, None])
    return _plain_grads(s, p, x, w, loss)


def _plain_kd(s):
    x, w, temp = s["x"].float(), s["weight"].float(), s["temp"]
    keep = s["ttokens"] >= 0
    valid = keep.any(dim=1)
    col = torch.where(keep, s["ttokens"], 0)
    tl = torch.where(keep, s["tlogits"] / temp, -1e30)
    eq = torch.exp(tl - tl.max(dim=1, keepdim=True).values) * keep
    q = eq / torch.where(valid, eq.sum(dim=1), 1.0)[:, None]
    z = (x @ w.t()).div_(temp)
    top = z.max(dim=1, keepdim=True).values
    zk = z.gather(1, col)
    e = torch.exp(z - top)
    total = e.sum(dim=1, keepdim=True)
    logq = torch.log(torch.where(q > 0, q, 1.0))
    loss = temp * temp * (q * (logq - (zk - top - torch.log(total)))).sum(dim=1)
    loss, share = _reduced(s, torch.where(valid, loss, 0.0), valid)
    if not s["grad"]:
        return {"loss": loss}
    p = e.div_(total)
    p.scatter_add_(1, col, -q)
    p.mul_((share * valid * temp)[:, None])
    return _plain_grads(s, p, x, w, loss)


# ---------------------------------------------------------------- the definitions, 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_embed(s) if case["op"] == "embed" else _exact_loss(s)


def _exact_embed(s):
    def rows(index, table):
        return table.detach().double().index_select(0, index)

    def summed(index, values, count):
        order = torch.argsort(index, stable=True)
        running = torch.cumsum(values[order], dim=0)
        ends = torch.searchsorted(index[order], torch.arange(count, device="cuda"), right=True)
        upto = torch.cat([torch.zeros(1, values.shape[1], dtype=torch.float64, device="cuda"), running])[ends]
        return torch.diff(upto, dim=0, prepend=torch.zeros_like(upto[:1]))

    out = s["scale"] * rows(s["ids"], s["weight"])
    if s["pos"]:
        out += rows(s["positions"], s["pweight"])
    if not s["grad"]:
        return {"out": out}
    g = s["gout"].double()
    gw = s["scale"] * summed(s["ids"], g, s["v"])
    if s["padding"] is not None:
        gw[s["padding"]] = 0.0
    grads = (gw, summed(s["positions"], g, s["pos"])) if s["pos"] else (gw,)
    return {"out": out, "grads": grads}


def _exact_loss(s):
    """The losses as divergences from a distribution over the vocabulary: all on the target, or the teacher's."""
    n, temp = s["n"], s.get("temp", 1.0)
    if s["op"] == "ce":
        tokens = s["targets"].clamp(min=0)[:, None]
        q = (s["targets"] != IGNORED).double()[:, None]
    else:
        tokens = s["ttokens"].clamp(min=0)
        t = s["tlogits"].double().div(temp).masked_fill(s["ttokens"] < 0, -math.inf)
        q = torch.nan_to_num(torch.softmax(t, dim=1), nan=0.0)
    valid = q.sum(dim=1) > 0
    x, w = s["x"].detach().double(), s["weight"].detach().double()
    count = valid.sum().double()
    losses, dxs, dw = [], [], torch.zeros_like(w)
    for at in range(0, n, 8192):                         # 3 GB of logits at a time
        sl = slice(at, min(n, at + 8192))
        logp = torch.log_softmax(x[sl] @ w.t() / temp, dim=1)
        picked = torch.gather(logp, 1, tokens[sl])
        loss = temp * temp * (torch.special.xlogy(q[sl], q[sl]) - q[sl] * picked).sum(dim=1)
        losses.append(torch.where(valid[sl], loss, 0.0))
        if s["grad"]:
            share = s["gout"][sl].double() if s["reduction"] == "none" else torch.ones_like(loss) if s["reduction"] == "sum" else torch.ones_like(loss) / count.clamp(min=1)
            dz = logp.exp_().scatter_add_(1, tokens[sl], -q[sl]) * (temp * share * valid[sl])[:, None]
            dxs.append(dz @ w)
            dw += dz.t() @ x[sl]
    loss = torch.cat(losses)
    loss = loss if s["reduction"] == "none" else loss.sum() if s["reduction"] == "sum" else loss.sum() / count.clamp(min=1)
    return {"loss": loss, "dx": torch.cat(dxs), "dw": dw} if s["grad"] else {"loss": loss}


def work(case):
    n, v, d = case["n"], case["v"], case["d"]
    if case["op"] == "embed":
        b, tables = BYTES[case["dtype"]], 1 + (case["pos"] > 0)
        touched = min(n, v) + min(n, case["pos"])
        moved = touched * d * b + n * d * b + 8 * n * tables
        if case["grad"]:
            moved += n * d * b + (v + case["pos"]) * d * b
        return {"bytes": moved, "flops": n * d * (2 if not case["grad"] else 4)}
    # the product once, and with gradients the two products that they are; rows, table, targets, results once each
    entries = n * (8 if case["op"] == "ce" else 12 * case["k"])
    moved = 2 * (n + v) * d + entries + (4 * n if case["reduction"] == "none" else 4)
    return {"bytes": moved + (2 * (n + v) * d if case["grad"] else 0), "flops": 2 * n * v * d * (3 if case["grad"] else 1)}
