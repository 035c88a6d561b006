"""Cross entropy and distillation over a vocabulary without the logits, against 64 bits.

What may be off, by arithmetic: a logit of d terms is added up in fp32 in steps of 16, each at most one step of its type (2**-23 of the
magnitudes' sum) off; a power of two or logarithm is a few of those; a gradient of a logit is rounded once to bf16 (2**-8 at most, less
than 2**-9 in the 2-norm over many), the gradients of x and weight once more."""
import pathlib
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

LN = 2.0 ** -18                      # of a loss's own size: powers, logarithms and sums in fp32


def logit_error(x, w):
    """Of every logit, [n, v]; with the largest of a row below."""
    return (x.shape[1] / 16 + 4) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t())


def problem(n, v, d, seed, spread=0.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, d, generator=gen, device="cuda").to(torch.bfloat16)
    w = (torch.randn(v, d, generator=gen, device="cuda") * (spread * 4 / d ** 0.5)).to(torch.bfloat16)
    return x, w, gen


def reference(x, w, tokens, q, temp):
    """Row losses, gradient of the logits for a gradient of 1 of each row's loss, logits' errors; q [n, k] weights of the entries."""
    z = x.double() @ w.double().t() / temp
    logp = torch.log_softmax(z, dim=1)
    keep = q > 0
    picked = logp.gather(1, torch.where(keep, tokens, 0))
    loss = temp * temp * torch.where(keep, torch.special.xlogy(q, q) - q * picked, 0.0).sum(dim=1)
    dz = temp * (logp.exp() * q.sum(dim=1, keepdim=True)).scatter_add(1, torch.where(keep, tokens, 0), -q)
    return loss, torch.where(keep.any(dim=1)[:, None], dz, 0.0)


def check_gradients(got, x, w, dz, share, temp, limit=2.0 ** -8, more=0.0):
    """Elementwise by the sums of magnitudes, and in the 2-norm: two roundings, each below 2**-9, are below 2**-8 together.
    ``more``: of a probability, in the gradient of w."""
    err = logit_error(x, w)
    rel = 2.0 ** -8 * (1 + 2.0 ** -8) + 2.0 ** -18 + 3 * err.max().item() / temp      # of p; p - q and its factor are rounded after it
    dz = dz * share[:, None]
    p = temp * share.abs()[:, None] * torch.softmax(x.double() @ w.double().t() / temp, dim=1)
    off = dz.abs() * rel + p * (rel - 2.0 ** -8)
    xd, wd = x.double(), w.double()
    depth = (max(x.shape[0], w.shape[0]) / 16 + 8) * 2.0 ** -23
    # a probability below the smallest normal number, 2**-126, is 0: of every term of a sum that much times the other factor
    least = 2.0 ** -126 * max(1.0, temp * share.abs().max().item())
    for name, g, want, bound, size in (("dx", got[0], dz @ wd, off @ wd.abs() + least * wd.abs().sum(dim=0), dz.abs() @ wd.abs()),
                                       ("dw", got[1], dz.t() @ xd, (off + more * p).t() @ xd.abs() + least * xd.abs().sum(dim=0), dz.abs().t() @ xd.abs())):
        if g is None:
            continue
        tol = bound * (1 + 2.0 ** -8) + want.abs() * 2.0 ** -8 + size * depth + 1e-38
        assert bool(((g.double() - want).abs() <= tol).all()), name
        norm = want.norm().item()
        if norm > 0 and want.numel() >= 4096:
            assert (g.double() - want).norm().item() <= limit * norm, name


def check_loss(got, want, x, w, temp):
    err = 2 * temp * logit_error(x, w).amax(dim=1)
    assert bool(((got.double() - want).abs() <= err + LN * (want.abs() + temp * temp)).all())


SIZES = [(1, 1, 8), (1, 2, 8), (1, 300, 16), (3, 257, 40), (77, 1000, 64), (128, 255, 72), (129, 256, 128), (255, 512, 136), (256, 513, 256), (257, 769, 264),
         (300, 5000, 200), (1000, 3001, 320), (2049, 640, 1024), (33, 50257, 64), (2, 50257, 768)]


@pytest.mark.parametrize("n,v,d", SIZES)
def test_cross_entropy(n, v, d):
    from dfccl_b200.ops.gemm import check_kernels
    from dfccl_b200.ops.loss import linear_cross_entropy
    x, w, gen = problem(n, v, d, n + 3 * v + 5 * d)
    t = torch.randint(0, v, (n,), generator=gen, device="cuda")
    drop = torch.rand(n, generator=gen, device="cuda") < 0.2
    drop[0] = False
    targets = torch.where(drop, -100, t)
    loss, dz = reference(x, w, t[:, None], (~drop).double()[:, None], 1.0)
    count = (~drop).sum().double()
    x.requires_grad_(True), w.requires_grad_(True)
    rows = linear_cross_entropy(x, w, targets, reduction="none")
    check_loss(rows.detach(), loss, x.detach(), w.detach(), 1.0)
    gout = torch.randn(n, generator=gen, device="cuda")
    check_gradients(torch.autograd.grad(rows, [x, w], gout), x.detach(), w.detach(), dz, gout.double(), 1.0)
    mean = linear_cross_entropy(x, w, targets)
    assert abs(mean.item() - (loss.sum() / count).item()) <= (2 * logit_error(x.detach(), w.detach()).max().item() + 2 * LN * (1 + loss.abs().max().item()))
    got = torch.autograd.grad(mean, [x, w], retain_graph=True)
    check_gradients(got, x.detach(), w.detach(), dz, torch.ones(n, device="cuda").double() / count, 1.0)
    again = torch.autograd.grad(mean, [x, w])
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    assert check_kernels()


@pytest.mark.parametrize("form", ["two", "one go", "one go in pieces"])
@pytest.mark.parametrize("n,v,d,k,temp", [(1, 1, 8, 1, 1.0), (1, 300, 16, 5, 2.0), (77, 1000, 64, 1, 0.5), (130, 515, 72, 32, 1.0), (257, 2049, 264, 33, 3.0),
                                          (300, 256, 128, 256, 2.0), (500, 5001, 320, 100, 1.5), (33, 50257, 64, 64, 1.0)])
def test_distillation(n, v, d, k, temp, form, monkeypatch):
    from dfccl_b200.ops import loss as module
    from dfccl_b200.ops.loss import linear_distillation
    monkeypatch.setattr(module, "ONE_GO_FROM", 1 << 60 if form == "two" else 0)
    monkeypatch.setattr(module, "LIST_SHARE", 0)
    if form == "one go in pieces":
        monkeypatch.setenv("DFCCL_LOSS_WORKSPACE_BYTES", str(1 << 20))
    x, w, gen = problem(n, v, d, n + 3 * v + 5 * d + k)
    tokens = torch.randint(0, v, (n, k), generator=gen, device="cuda")           # in any order, some twice
    logits = torch.randn(n, k, generator=gen, device="cuda") * 3
    tokens = torch.where(torch.rand(n, k, generator=gen, device="cuda") < 0.2, -1, tokens)
    tokens[n // 2] = -1 if n > 1 else tokens[0]
    logits = torch.where(torch.rand(n, k, generator=gen, device="cuda") < 0.05, float("-inf"), logits)
    keep = (tokens >= 0) & (logits > float("-inf"))
    valid = keep.any(dim=1)
    q = torch.nan_to_num(torch.softmax((logits.double() / temp).masked_fill(~keep, float("-inf")), dim=1), nan=0.0)
    loss, dz = reference(x, w, tokens.clamp(min=0), q, temp)
    x.requires_grad_(True), w.requires_grad_(True)
    rows = linear_distillation(x, w, torch.where(tokens < 0, float("nan"), logits), tokens, temperature=temp, reduction="none")
    check_loss(rows.detach(), loss, x.detach(), w.detach(), temp)
    assert bool((rows.detach()[~valid] == 0).all())
    gout = torch.randn(n, generator=gen, device="cuda")
    check_gradients(torch.autograd.grad(rows, [x, w], gout), x.detach(), w.detach(), dz, gout.double(), temp)
    total = linear_distillation(x, w, logits.to(torch.float32), tokens.int(), temperature=temp)
    mean = loss.sum().item() / max(1, int(valid.sum()))
    assert abs(total.item() - mean) <= 2 * temp * logit_error(x.detach(), w.detach()).max().item() + 2 * LN * (temp * temp + loss.abs().max().item())
    got = torch.autograd.grad(total, [x, w])
    check_gradients(got, x.detach(), w.detach(), dz, torch.ones(n, device="cuda").double() / max(1, int(valid.sum())), temp, more=0.0 if form == "two" else 2.0 ** -8 * (1 + 2.0 ** -8))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_teacher_types(dtype):
    """A list's order does not matter, and logits of 16 bits are what they are in 32."""
    from dfccl_b200.ops.loss import linear_distillation
    x, w, gen = problem(100, 700, 64, 5)
    tokens = torch.rand(100, 700, generator=gen, device="cuda").topk(24, dim=1).indices
    logits = torch.randn(100, 24, generator=gen, device="cuda").to(dtype)
    want = linear_distillation(x, w, logits.float(), tokens, reduction="none")
    assert torch.equal(want, linear_distillation(x, w, logits, tokens, reduction="none"))
    turned = linear_distillation(x, w, logits.flip(1), tokens.flip(1).int(), reduction="none")
    assert bool(((turned - want).abs() <= LN * (1 + want.abs())).all())          # the teacher's softmax adds up in the order of the list


@pytest.mark.parametrize("limit", [1 << 20, 3 << 20, 1 << 30])
@pytest.mark.parametrize("n,v,d", [(700, 5003, 128), (1500, 3000, 264), (100, 50257, 64)])
def test_pieces_of_the_vocabulary(n, v, d, limit, monkeypatch):
    """The gradient of the logits in one piece or many, with and without either of the two results."""
    from dfccl_b200.ops.loss import linear_cross_entropy
    monkeypatch.setenv("DFCCL_LOSS_WORKSPACE_BYTES", str(limit))
    x, w, gen = problem(n, v, d, n + v + d)
    t = torch.randint(0, v, (n,), generator=gen, device="cuda")
    _, dz = reference(x, w, t[:, None], torch.ones(n, 1, dtype=torch.float64, device="cuda"), 1.0)
    for want_x, want_w in ((True, True), (True, False), (False, True)):
        xl, wl = x.clone().requires_grad_(want_x), w.clone().requires_grad_(want_w)
        linear_cross_entropy(xl, wl, t, reduction="sum").backward()
        check_gradients((xl.grad, wl.grad), x, w, dz, torch.ones(n, dtype=torch.float64, device="cuda"), 1.0)


ONE_GO = [(1, 1, 8), (1, 300, 16), (77, 1000, 64), (255, 513, 136), (256, 512, 256), (300, 5000, 200), (1000, 3001, 320), (2049, 640, 1024), (40, 50257, 64)]


@pytest.mark.parametrize("limit", [1 << 20, 1 << 30])
@pytest.mark.parametrize("n,v,d", ONE_GO)
def test_gradients_with_the_loss(n, v, d, limit, monkeypatch):
    """The form that large losses take, in one piece of rows or several: the powers are rounded once for both gradients (the target's share of
    them is not), and x times a row's share once more for that of w.  Scaled by what comes from behind, one more rounding."""
    from dfccl_b200.ops import loss as module
    from dfccl_b200.ops.gemm import check_kernels
    monkeypatch.setattr(module, "ONE_GO_FROM", 0)
    monkeypatch.setenv("DFCCL_LOSS_WORKSPACE_BYTES", str(limit))
    x, w, gen = problem(n, v, d, n + 3 * v + 5 * d)
    t = torch.randint(0, v, (n,), generator=gen, device="cuda")
    drop = torch.rand(n, generator=gen, device="cuda") < 0.2
    drop[0] = False
    targets = torch.where(drop, -100, t)
    loss, dz = reference(x, w, t[:, None], (~drop).double()[:, None], 1.0)
    count = (~drop).sum().double()
    two = 2.0 ** -8 * (1 + 2.0 ** -8)
    for reduction, share in (("mean", 1.0 / count), ("sum", torch.ones_like(count))):
        for want_x, want_w in ((True, True), (True, False), (False, True)):
            a, b = x.clone().requires_grad_(want_x), w.clone().requires_grad_(want_w)
            value = module.linear_cross_entropy(a, b, targets, reduction=reduction)
            err = 2 * logit_error(x, w).max().item() + 2 * LN * (1 + loss.abs().max().item())
            assert abs(value.item() - (loss.sum() * share).item()) <= err * (1 if reduction == "mean" else n)
            value.backward(retain_graph=True)
            each = share.expand(n)
            check_gradients((a.grad, b.grad), x, w, dz, each, 1.0, more=two)
            first = [None if g is None else g.clone() for g in (a.grad, b.grad)]
            a.grad = b.grad = None
            (value * 3).backward()                       # the same graph again: the logits are computed again
            check_gradients((a.grad, b.grad), x, w, dz, 3 * each, 1.0)
            a.grad = b.grad = None
            other = module.linear_cross_entropy(a, b, targets, reduction=reduction)
            if want_x and want_w:                        # one after the other: the second is computed again
                pair = [torch.autograd.grad(other, [leaf], retain_graph=True)[0] for leaf in (a, b)]
                assert torch.equal(pair[0], first[0])
                check_gradients((None, pair[1]), x, w, dz, each, 1.0, more=two)
                other = module.linear_cross_entropy(a, b, targets, reduction=reduction)
            (other * 0.3).backward()
            for g, f in zip((a.grad, b.grad), first):    # one rounding of 0.3 times the same values
                if g is not None:
                    assert torch.equal(g, (f.float() * 0.3).to(torch.bfloat16))
    assert check_kernels()


def test_gradients_with_the_loss_of_odd_rows(monkeypatch):
    """Targets far below their row's largest logit (powers above 2**60, which send the piece through once more), ignored rows that hold
    anything, a target of probability one; infinities, NaN and targets outside give what they give otherwise."""
    from dfccl_b200.ops import loss as module
    monkeypatch.setattr(module, "ONE_GO_FROM", 0)
    n, v, d = 400, 900, 64
    for spread in (0.5, 40.0):
        x, w, gen = problem(n, v, d, 77, spread=spread)
        t = torch.randint(0, v, (n,), generator=gen, device="cuda")
        t[::7] = (x[::7].double() @ w.double().t()).argmax(dim=1)
        hole = torch.arange(n, device="cuda") % 5 == 2
        targets = torch.where(hole, -100, t)
        loss, dz = reference(x, w, t[:, None], (~hole).double()[:, None], 1.0)
        dirty = x.clone()
        dirty[hole] = torch.tensor([float("inf"), float("nan"), float("-inf"), 1e38], device="cuda").to(torch.bfloat16).repeat(16)
        a, b = dirty.clone().requires_grad_(True), w.clone().requires_grad_(True)
        value = module.linear_cross_entropy(a, b, targets, reduction="sum")
        assert abs(value.item() - loss.sum().item()) <= n * 2 * logit_error(x, w).max().item() + 2 * LN * (n + loss.sum().item())
        value.backward()
        a.grad[hole] += 0                                # (zeros stay)
        check_gradients((a.grad, b.grad), x, w, dz, torch.ones(n, device="cuda").double(), 1.0, more=2.0 ** -8)
        assert bool((a.grad[hole] == 0).all())
        # lists: the student nearly certain of an entry, or of none
        lists = torch.stack([t, (t + 1) % v, t], dim=1)
        teacher = torch.tensor([2.0, 1.0, 0.5], device="cuda").expand(n, 3)
        q = torch.softmax(teacher.double(), dim=1) * (~hole).double()[:, None]
        loss, dz = reference(x, w, lists, q, 1.0)
        a, b = dirty.clone().requires_grad_(True), w.clone().requires_grad_(True)
        monkeypatch.setattr(module, "LIST_SHARE", 0)
        value = module.linear_distillation(a, b, teacher, torch.where(hole[:, None], -1, lists), reduction="sum")
        assert abs(value.item() - loss.sum().item()) <= n * 2 * logit_error(x, w).max().item() + 2 * LN * (n + loss.sum().item())
        value.backward()
        check_gradients((a.grad, b.grad), x, w, dz, torch.ones(n, device="cuda").double(), 1.0, more=2.0 ** -8)
        assert bool((a.grad[hole] == 0).all())
    zero, b = dirty.clone().requires_grad_(True), w.clone().requires_grad_(True)
    value = module.linear_cross_entropy(zero, b, torch.full_like(t, -100))
    value.backward()
    assert value.item() == 0.0 and bool((zero.grad == 0).all()) and bool((b.grad == 0).all())
    for bad in (v, -1):
        a = x.clone().requires_grad_(True)
        value = module.linear_cross_entropy(a, w, torch.where(torch.arange(n, device="cuda") == 3, bad, t))
        value.backward()
        assert value.isnan().item() and a.grad.isnan().any(dim=1).nonzero()[:, 0].tolist() == [3]
    for k, value in ((8, float("-inf")), (9, float("inf")), (10, float("nan"))):
        w2, ones = w.clone(), torch.ones_like(x)
        w2[k] = value
        with torch.no_grad():
            plain = [module.linear_cross_entropy(ones, w2, torch.full_like(t, c), reduction="sum") for c in (k, 20)]
        odd = [module.linear_cross_entropy(ones.clone().requires_grad_(True), w2, torch.full_like(t, c), reduction="sum") for c in (k, 20)]
        for p, q in zip(plain, odd):
            assert torch.equal(p.isnan(), q.isnan()) and (p.isnan().item() or abs(p.item() - q.item()) <= 1e-5 * abs(p.item()) or p.item() == q.item())


@pytest.mark.parametrize("one_go", [False, True])
@pytest.mark.parametrize("n", [3, 5000])
def test_gradients_of_nearly_certain_rows(n, one_go, monkeypatch):
    """Rows whose target has all but 1e-4 of the probability: their gradients are that small, and as exact as any other."""
    from dfccl_b200.ops import loss as module
    monkeypatch.setattr(module, "ONE_GO_FROM", 0 if one_go else 1 << 60)
    monkeypatch.setattr(module, "LIST_SHARE", 0)
    v, d = 300, 64
    gen = torch.Generator(device="cuda").manual_seed(61)
    w = (torch.randn(v, d, generator=gen, device="cuda") * 0.05).to(torch.bfloat16)
    t = torch.randint(0, v, (n,), generator=gen, device="cuda")
    wt = w[t].float()
    x = (torch.randn(n, d, generator=gen, device="cuda") * 0.2 + wt * (14.5 / wt.square().sum(dim=1, keepdim=True))).to(torch.bfloat16)
    loss, dz = reference(x, w, t[:, None], torch.ones(n, 1, dtype=torch.float64, device="cuda"), 1.0)
    assert 2e-6 < loss.median().item() < 1e-2
    for call in (lambda a, b: module.linear_cross_entropy(a, b, t), lambda a, b: module.linear_distillation(a, b, torch.zeros(n, 1, device="cuda"), t[:, None])):
        a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        value = call(a, b)
        # logits of 15 and less, off by 2**-20: of the others' powers, and so of the loss and all gradients, that share
        assert abs(value.item() - loss.mean().item()) <= 2.0 ** -18 * loss.mean().item()
        ga, gb = torch.autograd.grad(value, [a, b])
        for got, want in ((ga, dz @ w.double() / n), (gb, dz.t() @ x.double() / n)):
            # a rounding of the result, and of x times a row's share beside the others' powers: below 2**-9 and 2**-8 in the 2-norm
            assert (got.double() - want).norm().item() <= 2.0 ** -8 * 1.5 * want.norm().item()


def test_small_losses_and_large_logits():
    """The logits of the targets are not what the tensor cores cut off, whichever way the loss goes: rows whose target stands out by 20, from
    2048 products of one sign, have a loss of 2e-9 relative to 900 others, and those of the others one of 20."""
    from dfccl_b200.ops.loss import linear_cross_entropy, linear_distillation
    n, v, d = 64, 900, 2048
    w = torch.zeros(v, d, device="cuda", dtype=torch.bfloat16)
    w[5] = 2.0 ** -7
    x = torch.full((n, d), 1.25, device="cuda", dtype=torch.bfloat16)            # logits of 20 exactly, and of 0
    for token, want in ((5, 899 * 2.061153622438558e-09), (6, 20 + 899 * 2.061153622438558e-09)):
        t = torch.full((n,), token, device="cuda")
        got = linear_cross_entropy(x, w, t, reduction="none").double()
        assert bool(((got - want).abs() <= 2.0 ** -22 * 20 + 2.0 ** -22).all())
        again = linear_distillation(x, w, torch.zeros(n, 1, device="cuda"), t[:, None], reduction="none")
        assert bool(((again.double() - want).abs() <= 2.0 ** -22 * 20 + 2.0 ** -22).all())


def test_ignored_rows_hold_anything():
    """Infinities and NaN in rows without a target reach nothing; a batch without any target costs nothing and gives zeros."""
    from dfccl_b200.ops.loss import linear_cross_entropy, linear_distillation
    x, w, gen = problem(300, 1000, 64, 9)
    t = torch.randint(0, 1000, (300,), generator=gen, device="cuda")
    hole = torch.arange(300, device="cuda") % 3 == 1
    dirty = x.clone()
    dirty[hole] = torch.tensor([float("inf"), float("nan"), float("-inf"), 1e38], device="cuda").to(torch.bfloat16).repeat(16)
    t = torch.where(hole, -100, t)
    lists = torch.where(hole[:, None], -1, torch.stack([t, (t + 1) % 1000], dim=1))
    teacher = torch.zeros(300, 2, device="cuda")
    for loss in (lambda a, b: linear_cross_entropy(a, b, t), lambda a, b: linear_distillation(a, b, teacher, lists)):
        res = []
        for rows in (x, dirty):
            a, b = rows.clone().requires_grad_(True), w.clone().requires_grad_(True)
            value = loss(a, b)
            value.backward()
            res.append((value.detach(), a.grad, b.grad))
        clean, mixed = res
        assert torch.equal(clean[0], mixed[0])
        assert torch.equal(clean[1][~hole], mixed[1][~hole]) and bool((mixed[1][hole] == 0).all())
        # the rows' zeros stand beside x's NaN in the product of the weight's gradient: they must not meet
        assert torch.equal(clean[2], mixed[2])
    a, b = dirty.clone().requires_grad_(True), w.clone().requires_grad_(True)
    for value in (linear_cross_entropy(a, b, torch.full_like(t, -100)), linear_distillation(a, b, teacher, torch.full_like(lists, -1))):
        assert value.item() == 0.0
        ga, gb = torch.autograd.grad(value, [a, b])
        assert bool((ga == 0).all()) and bool((gb == 0).all())


def test_large_and_infinite_logits():
    """Logits of hundreds, a head with a row of the type's lowest value or of -inf logits, equal logits; a row of NaN is NaN by itself."""
    from dfccl_b200.ops.loss import linear_cross_entropy
    x, w, gen = problem(200, 900, 64, 21, spread=40.0)
    t = torch.randint(0, 900, (200,), generator=gen, device="cuda")
    loss, dz = reference(x, w, t[:, None], torch.ones(200, 1, dtype=torch.float64, device="cuda"), 1.0)
    rows = linear_cross_entropy(x, w, t, reduction="none")
    check_loss(rows, loss, x, w, 1.0)
    ones = torch.ones(200, 64, device="cuda").to(torch.bfloat16)
    w2 = w.clone()
    w2[7] = torch.finfo(torch.bfloat16).min / 128
    w2[8] = float("-inf")
    t = torch.where((t == 7) | (t == 8), 9, t)
    got = linear_cross_entropy(ones, w2, t, reduction="none")
    kept = torch.cat([w[:7], w[9:]])
    want, _ = reference(ones, kept, torch.where(t > 8, t - 2, t)[:, None], torch.ones(200, 1, dtype=torch.float64, device="cuda"), 1.0)
    check_loss(got, want, ones, kept, 1.0)
    assert linear_cross_entropy(ones[:1], w2, torch.tensor([8], device="cuda")).item() == float("inf")
    flat = linear_cross_entropy(ones, torch.zeros_like(w), t, reduction="none")
    assert bool(((flat - torch.log(torch.tensor(900.0))).abs() < 1e-5).all())
    x[5, 3] = float("nan")
    rows = linear_cross_entropy(x, w, t, reduction="none")
    assert rows.isnan().nonzero()[:, 0].tolist() == [5]


def test_targets_outside_the_vocabulary():
    from dfccl_b200.ops.loss import linear_cross_entropy, linear_distillation
    x, w, gen = problem(64, 300, 32, 23)
    t = torch.randint(0, 300, (64,), generator=gen, device="cuda")
    t[3], t[40], t[50] = 300, -1, 2 ** 33
    rows = linear_cross_entropy(x, w, t, reduction="none")
    assert rows.isnan().nonzero()[:, 0].tolist() == [3, 40, 50]
    lists = t[:, None].clamp(min=-1)
    lists[41] = -2
    rows = linear_distillation(x, w, torch.zeros(64, 1, device="cuda"), lists, reduction="none")
    assert rows.isnan().nonzero()[:, 0].tolist() == [3, 41, 50] and rows[40].item() == 0.0
    a = x.clone().requires_grad_(True)
    linear_distillation(a, w, torch.zeros(64, 1, device="cuda"), lists, reduction="sum").backward()
    assert a.grad.isnan().any(dim=1).nonzero()[:, 0].tolist() == [3, 41, 50]


def test_strides_shapes_and_gradients_of_one_value():
    from dfccl_b200.ops.loss import linear_cross_entropy
    x, w, gen = problem(60, 500, 72, 31)
    t = torch.randint(0, 500, (60,), generator=gen, device="cuda")
    want = linear_cross_entropy(x, w, t, reduction="none")
    wide = torch.zeros(60, 80, device="cuda", dtype=torch.bfloat16)
    wide[:, 3:75] = x
    assert torch.equal(want, linear_cross_entropy(wide[:, 3:75], w.t().contiguous().t(), t.int(), reduction="none"))
    shaped = linear_cross_entropy(x.view(3, 20, 72), w, t.view(3, 20), reduction="none")
    assert shaped.shape == (3, 20) and torch.equal(shaped.view(-1), want)
    a, b = wide.clone().requires_grad_(True), w.clone().requires_grad_(True)
    linear_cross_entropy(a[:, 3:75].view(4, 15, 72), b, t.view(4, 15), reduction="none").sum().backward()
    c, d = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    linear_cross_entropy(c, d, t, reduction="sum").backward()
    assert torch.equal(a.grad[:, 3:75], c.grad) and torch.equal(b.grad, d.grad) and bool((a.grad[:, :3] == 0).all())
    none = linear_cross_entropy(x[:0].requires_grad_(True), d, t[:0])
    assert none.item() == 0.0
    assert bool((torch.autograd.grad(none, [d])[0] == 0).all())
    one = linear_cross_entropy(x[0], w, t[0], reduction="none")
    assert one.shape == () and torch.equal(one, want[0])


def test_gradient_against_differences():
    """The loss, in 64 bits, along the gradient: central differences of the reference against what the kernels give."""
    from dfccl_b200.ops.loss import linear_cross_entropy
    x, w, gen = problem(96, 700, 64, 37)
    t = torch.randint(0, 700, (96,), generator=gen, device="cuda")
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    ga, gb = torch.autograd.grad(linear_cross_entropy(a, b, t), [a, b])

    def value(step):
        z = (x.double() + step * ga.double()) @ (w.double() + step * gb.double()).t()
        return torch.nn.functional.cross_entropy(z, t).item()

    slope = (value(1e-4) - value(-1e-4)) / 2e-4
    size = (ga.double().square().sum() + gb.double().square().sum()).item()
    assert abs(slope - size) <= 2.0 ** -8 * size                      # the gradients' error in the 2-norm, along themselves


@pytest.mark.parametrize("one_go", [False, True])
def test_other_stream_and_graphs(one_go, monkeypatch):
    """On a stream of its own; forward and backward captured and replayed for other data, two graphs in turns."""
    from dfccl_b200.ops import loss as module
    from dfccl_b200.ops.gemm import check_kernels
    from dfccl_b200.ops.loss import linear_cross_entropy, linear_distillation
    monkeypatch.setattr(module, "ONE_GO_FROM", 0 if one_go else 1 << 60)
    monkeypatch.setattr(module, "LIST_SHARE", 0)
    x, w, gen = problem(300, 3001, 128, 41)
    w.requires_grad_(True)
    xs = [torch.randn(300, 128, generator=gen, device="cuda").to(torch.bfloat16) for _ in range(3)]
    ts = [torch.randint(-1, 3001, (300, 4), generator=gen, device="cuda") for _ in range(3)]
    teacher = torch.randn(300, 4, generator=gen, device="cuda")

    def step(x, t):
        x = x.detach().requires_grad_(True)
        loss = linear_cross_entropy(x, w, t[:, 0], ignore_index=-1) + linear_distillation(x, w, teacher, t, temperature=2.0)
        return (loss.detach(),) + torch.autograd.grad(loss, [x, w])

    want = [step(a, b) for a, b in zip(xs, ts)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(xs[1], ts[1])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[1]))
    graphs = []
    for _ in range(2):
        a, b = xs[0].clone(), ts[0].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(a, b)
        graphs.append((a, b, graph, out))
    for turn in range(3):
        for k, (a, b, graph, _) in enumerate(graphs):
            a.copy_(xs[(turn + k) % 3]), b.copy_(ts[(turn + k) % 3])
            graph.replay()
        for k, (_, _, _, out) in enumerate(graphs):
            assert all(torch.equal(p, q) for p, q in zip(out, want[(turn + k) % 3]))
    assert check_kernels()


@pytest.mark.parametrize("one_go", [False, True])
@pytest.mark.parametrize("lists", [False, True])
def test_one_gradient_of_two(lists, one_go, monkeypatch):
    """A frozen head, or inputs that want no gradient: the other gradient is the same."""
    from dfccl_b200.ops import loss as module
    from dfccl_b200.ops.loss import linear_cross_entropy, linear_distillation
    monkeypatch.setattr(module, "ONE_GO_FROM", 0 if one_go else 1 << 60)
    monkeypatch.setattr(module, "LIST_SHARE", 0)
    for n, v, d, k in ((3, 700, 64, 2), (300, 3001, 136, 20)):
        x, w, gen = problem(n, v, d, 61)
        t = torch.randint(0, v, (n, k), generator=gen, device="cuda")
        teacher = torch.randn(n, k, generator=gen, device="cuda")

        def gradients(want_x, want_w):
            a, b = x.clone().requires_grad_(want_x), w.clone().requires_grad_(want_w)
            loss = linear_distillation(a, b, teacher, t) if lists else linear_cross_entropy(a, b, t[:, 0])
            loss.backward()
            return a.grad, b.grad

        both, left, right = gradients(True, True), gradients(True, False), gradients(False, True)
        assert left[1] is None and right[0] is None
        for a, b in ((left[0], both[0]), (right[1], both[1])):     # (slices of the contraction may be cut elsewhere: results a rounding apart)
            assert bool(((a.double() - b.double()).abs() <= 2.0 ** -7 * b.double().abs() + 1e-6 * b.double().abs().max()).all())


@pytest.mark.parametrize("one_go", [False, True])
def test_no_rows(one_go, monkeypatch):
    from dfccl_b200.ops import loss as module
    from dfccl_b200.ops.loss import linear_cross_entropy, linear_distillation
    monkeypatch.setattr(module, "ONE_GO_FROM", 0 if one_go else 1 << 60)
    monkeypatch.setattr(module, "LIST_SHARE", 0)
    x = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    w = torch.ones(300, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    none = torch.empty(0, 4, 2, dtype=torch.int64, device="cuda")
    for reduction in ("none", "sum", "mean"):
        for loss in (linear_cross_entropy(x, w, none[..., 0], reduction=reduction), linear_distillation(x, w, none.float(), none, reduction=reduction)):
            assert loss.shape == ((0, 4) if reduction == "none" else ()) and loss.sum().item() == 0.0
            dx, dw = torch.autograd.grad(loss.sum(), [x, w])
            assert dx.shape == x.shape and bool((dw == 0).all())


def test_first_backward_pass_of_a_process_with_a_frozen_head():
    """The thread of backward passes has made no call of the CUDA runtime yet."""
    code = """
import torch
from dfccl_b200.ops.loss import linear_cross_entropy
x = torch.randn(5, 64, device="cuda").to(torch.bfloat16).requires_grad_(True)
w = torch.randn(300, 64, device="cuda").to(torch.bfloat16)
torch.empty(1 << 24, device="cuda")
linear_cross_entropy(x, w, torch.arange(5, device="cuda")).backward()
assert x.grad.isfinite().all() and (x.grad != 0).any()
"""
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=pathlib.Path(__file__).parents[1])
    assert run.returncode == 0, run.stderr[-2000:]


@pytest.mark.parametrize("loss_captured", [False, True])
@pytest.mark.parametrize("lists", [False, True])
def test_backward_pass_captured_apart_from_the_loss(lists, loss_captured, monkeypatch):
    """Each replay of the pass gives the gradients of the loss, however often the same loss's pass is replayed."""
    from dfccl_b200.ops import loss as module
    from dfccl_b200.ops.gemm import check_kernels
    from dfccl_b200.ops.loss import linear_cross_entropy, linear_distillation
    monkeypatch.setattr(module, "ONE_GO_FROM", 0)
    monkeypatch.setattr(module, "LIST_SHARE", 0)
    x, w, gen = problem(300, 3001, 128, 51)
    x.requires_grad_(True), w.requires_grad_(True)
    t = torch.randint(0, 3001, (300, 4), generator=gen, device="cuda")
    teacher = torch.randn(300, 4, generator=gen, device="cuda")
    g = torch.full((), 3.0, device="cuda")

    def loss_of():
        return linear_distillation(x, w, teacher, t, temperature=2.0) if lists else linear_cross_entropy(x, w, t[:, 0])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss = loss_of()
        first = torch.autograd.grad(loss, [x, w], g, retain_graph=True)
        want = torch.autograd.grad(loss, [x, w], g)            # the logits computed again, as in the captured pass
        loss = None if loss_captured else loss_of()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, want):                              # (each: probabilities, and the result up to twice, rounded)
        assert (a.double() - b.double()).norm().item() <= 3 * 2.0 ** -8 * b.double().norm().item()
    graphs = []
    if loss_captured:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[0], stream=side):
            loss = loss_of()
    graphs.append(torch.cuda.CUDAGraph())
    with torch.cuda.graph(graphs[-1], stream=side, pool=graphs[0].pool() if loss_captured else None):
        got = torch.autograd.grad(loss, [x, w], g, retain_graph=True)
    graphs[0].replay()
    for _ in range(3):
        graphs[-1].replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert check_kernels()


def test_many_rows_and_wide_ones():
    """More rows than the statistics take at a time, a width of many stages, row numbers beyond 16 bits."""
    from dfccl_b200.ops.gemm import check_kernels
    from dfccl_b200.ops.loss import linear_cross_entropy, linear_distillation
    for n, v, d in ((40001, 300, 16), (16385, 40, 8), (70000, 9, 24), (130, 700, 8192)):
        x, w, gen = problem(n, v, d, n + v + d)
        t = torch.randint(0, v, (n,), generator=gen, device="cuda")
        t[n // 3] = -100
        keep = (t >= 0).double()[:, None]
        loss, dz = reference(x, w, t.clamp(min=0)[:, None], keep, 1.0)
        x.requires_grad_(True), w.requires_grad_(True)
        value = linear_cross_entropy(x, w, t, reduction="sum")
        err = 2 * logit_error(x.detach(), w.detach()).amax(dim=1).sum().item() + 2 * LN * (n + loss.sum().item())
        assert abs(value.item() - loss.sum().item()) <= err
        check_gradients(torch.autograd.grad(value, [x, w]), x.detach(), w.detach(), dz, torch.ones(n, device="cuda").double(), 1.0)
        rows = linear_distillation(x, w, torch.zeros(n, 1, device="cuda"), t.clamp(min=-1)[:, None], reduction="none")
        check_loss(rows.detach(), loss, x.detach(), w.detach(), 1.0)
    assert check_kernels()


@pytest.mark.parametrize("one_go", [False, True])
def test_a_head_of_more_elements_than_31_bits_count(one_go, monkeypatch):
    """The last rows of the vocabulary, where the offsets of w and of its gradient need 64 bits, and dx, which sums over all of it."""
    from dfccl_b200.ops import loss as module
    from dfccl_b200.ops.loss import linear_cross_entropy
    monkeypatch.setattr(module, "ONE_GO_FROM", 0 if one_go else 1 << 60)
    n, v, d, last = 40, 530003, 4096, 64
    gen = torch.Generator(device="cuda").manual_seed(71)
    x = torch.randn(n, d, generator=gen, device="cuda").to(torch.bfloat16).requires_grad_(True)
    w = (torch.randn(v, d, generator=gen, device="cuda", dtype=torch.bfloat16) * 0.03125).requires_grad_(True)
    t = torch.randint(0, v, (n,), generator=gen, device="cuda")
    t[::2] = v - 1 - torch.arange(n // 2, device="cuda")
    loss = linear_cross_entropy(x, w, t)
    dx, dw = torch.autograd.grad(loss, [x, w])
    xd, cuts = x.detach().double(), range(0, v, 65536)
    z = torch.cat([xd @ w.detach()[c:c + 65536].double().t() for c in cuts], dim=1)
    assert abs(loss.item() - torch.nn.functional.cross_entropy(z, t).item()) <= 1e-5 * loss.item()
    dz = torch.softmax(z, dim=1).scatter_add(1, t[:, None], torch.full((n, 1), -1.0, dtype=torch.float64, device="cuda")) / n
    want = sum(dz[:, c:c + 65536] @ w.detach()[c:c + 65536].double() for c in cuts)
    # (each result two roundings, as everywhere above)
    assert (dx.double() - want).norm() <= 2.0 ** -8 * want.norm()
    for rows in (slice(0, last), slice(v - last, v)):
        want = dz[:, rows].t() @ xd
        assert (dw[rows].double() - want).norm() <= 2.0 ** -8 * want.norm()


def test_calls_on_two_streams_at_once():
    """Two losses and an embedding on streams of their own, in flight together, each as by itself."""
    from dfccl_b200.ops.embedding import embedding
    from dfccl_b200.ops.loss import linear_cross_entropy
    data = []
    for k in range(2):
        x, w, gen = problem(600 + 100 * k, 4000, 256, 50 + k)
        data.append((x.requires_grad_(True), w.requires_grad_(True), torch.randint(0, 4000, (x.shape[0],), generator=gen, device="cuda")))

    def step(k):
        x, w, t = data[k]
        h = embedding(t, w)
        loss = linear_cross_entropy(x, w, t)
        return (h.detach(), loss.detach()) + torch.autograd.grad([loss, h], [x, w], [torch.ones((), device="cuda"), torch.ones_like(h)])

    want = [step(k) for k in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(5):
        got = []
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(step(k))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_a_models_two_ends():
    """A stage of GPT-2 with its ends on these kernels against the same weights without: the embedding's rows are the same, the loss is
    off by the rounding of the logits to bf16 (2**-9 of logits of a few units, over many rows), every gradient by roundings to bf16."""
    from dfccl_b200 import native as nv
    from dfccl_b200.models.gpt2 import GPT2Config, GPT2Stage
    from dfccl_b200.ops.fused_linear import TpGroup
    (comm,) = nv.Comm.init_loopback(1, torch.cuda.current_device())
    cfg = GPT2Config(n_layer=1, d_model=256, n_head=4, seq_len=128, vocab=1111)
    tp = TpGroup(comm, None, torch.device("cuda", torch.cuda.current_device()))
    plain, fused = GPT2Stage(cfg, tp, 0, 1, 4), GPT2Stage(cfg, tp, 0, 1, 4, fused_ends=True)
    tokens = torch.randint(0, 1111, (4, 129), device="cuda")
    losses, grads = [], []
    for stage in (plain, fused):
        loss = stage(tokens[:, :-1], tokens[:, 1:])
        loss.backward()
        losses.append(loss.item())
        grads.append([p.grad.double() for p in stage.parameters()])
    assert abs(losses[0] - losses[1]) <= 2.0 ** -9 * losses[0]
    for a, b in zip(*grads):
        assert (a - b).norm().item() <= 0.03 * a.norm().item()       # several roundings of 2**-9 on either side, through a block
    comm.destroy()


def certain_lists(n, v, d, k, seed):
    """Rows whose lists' tokens have all but some 1e-4 of the student's probability, and a teacher who weighs them differently: what the lists
    add is nearly all of both gradients.  Returns x, w, tokens, teacher's logits."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    w = (torch.randn(v, d, generator=gen, device="cuda") * 0.05).to(torch.bfloat16)
    tokens = torch.rand(n, v, generator=gen, device="cuda").topk(k, dim=1).indices
    # the smallest x with a logit of 15 for each of the row's tokens
    wt = w[tokens].double()
    x = (wt.transpose(1, 2) @ torch.linalg.inv(wt @ wt.transpose(1, 2)) @ torch.full((n, k, 1), 15.0, dtype=torch.float64, device="cuda"))[..., 0]
    return x.to(torch.bfloat16), w, tokens, torch.randn(n, k, generator=gen, device="cuda")


def check_lists(got, x, w, tokens, q, share, temp=1.0):
    """Against 64 bits, element by element: half a step of the result, half a step of bf16 (2**-8) for the probabilities of what stands in no list, and
    fp32 for the lists' own, which are q less a probability."""
    loss, dz = reference(x, w, tokens, q, temp)
    dz = dz * share[:, None]
    err = 3 * logit_error(x, w).max().item() / temp + 2.0 ** -18             # of a probability, relative
    p = temp * share.abs()[:, None] * torch.softmax(x.double() @ w.double().t() / temp, dim=1)
    listed = torch.zeros_like(dz).scatter_(1, tokens, 1.0)
    off = p * err + torch.where(listed > 0, 2.0 ** -22 * temp * share.abs()[:, None], p * 2.0 ** -8 * (1 + 2.0 ** -8))
    xd, wd = x.double(), w.double()
    depth = (max(dz.shape) / 16 + 8) * 2.0 ** -23
    for name, g, want, bound, size in (("dx", got[0], dz @ wd, off @ wd.abs(), dz.abs() @ wd.abs()),
                                       ("dw", got[1], dz.t() @ xd, off.t() @ xd.abs(), dz.abs().t() @ xd.abs())):
        if g is not None:
            assert bool(((g.double() - want).abs() <= bound * (1 + 2.0 ** -8) + want.abs() * 2.0 ** -8 + size * depth + 1e-38).all()), name
    return loss


# entries below and above 2048, below and above the vocabulary, lists that fit the products' epilogue and longer ones
@pytest.mark.parametrize("n,v,d,k", [(500, 300, 64, 3), (700, 300, 64, 3), (700, 300, 64, 7), (800, 4001, 128, 3), (300, 4001, 136, 9), (2500, 257, 264, 4)])
@pytest.mark.parametrize("limit", [1 << 20, 1 << 30])
def test_what_lists_add_keeps_its_digits(n, v, d, k, limit, monkeypatch):
    """Whichever way the loss goes, however many entries there are, in one piece of the vocabulary or several."""
    from dfccl_b200.ops import loss as module
    from dfccl_b200.ops.gemm import check_kernels
    monkeypatch.setenv("DFCCL_LOSS_WORKSPACE_BYTES", str(limit))
    monkeypatch.setattr(module, "ONE_GO_FROM", 1 << 60)
    x, w, tokens, teacher = certain_lists(n, v, d, k, n + v + d + k)
    hole = torch.arange(n, device="cuda") % 9 == 4
    q = torch.softmax(teacher.double(), dim=1) * (~hole).double()[:, None]
    given = torch.where(hole[:, None], -1, tokens)
    gout = torch.randn(n, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    for want_x, want_w in ((True, True), (True, False), (False, True)):
        a, b = x.clone().requires_grad_(want_x), w.clone().requires_grad_(want_w)
        rows = module.linear_distillation(a, b, teacher, given, reduction="none")
        rows.backward(gout)
        loss = check_lists((a.grad, b.grad), x, w, tokens, q, gout.double())
        check_loss(rows.detach(), loss, x, w, 1.0)
        a.grad = b.grad = None
        module.linear_distillation(a, b, teacher, given).backward()
        check_lists((a.grad, b.grad), x, w, tokens, q, torch.full((n,), 1.0 / int((~hole).sum()), dtype=torch.float64, device="cuda"))
    assert check_kernels()


def test_coldest_and_hottest_teachers():
    """The ends of the temperatures: at 2**-20 logits of +-300 are exponents of 4e8, which fp32 tells apart by 32; at 2**20 the loss, some units, is what a
    few roundings leave of T^2 = 1e12: only its gradient is of use."""
    from dfccl_b200.ops.loss import linear_distillation
    n, v, d = 100, 600, 64
    x, w, gen = problem(n, v, d, 3, spread=4.0)
    t = torch.randint(0, v, (n, 3), generator=gen, device="cuda")
    t[:, 1], t[:, 2] = (t[:, 0] + 1) % v, (t[:, 0] + 2) % v
    teacher = torch.randn(n, 3, generator=gen, device="cuda")
    for temp in (2.0 ** -20, 2.0 ** 20):
        q = torch.softmax(teacher.double() / temp, dim=1)
        loss, dz = reference(x, w, t, q, temp)
        a = x.clone().requires_grad_(True)
        rows = linear_distillation(a, w, teacher, t, temperature=temp, reduction="none")
        rows.sum().backward()
        err = 2 * temp * logit_error(x, w).amax(dim=1) + 2.0 ** -22 * 3 * temp * (x.double() @ w.double().t()).abs().amax(dim=1)
        assert bool(((rows.detach().double() - loss).abs() <= err + LN * (loss.abs() + temp * temp)).all())
        assert a.grad.isfinite().all()
        if temp > 1:                                     # (at 2**-20 a logit's error is a thousand steps of an exponent)
            assert (a.grad.double() - dz @ w.double()).norm() <= 2.0 ** -8 * (dz @ w.double()).norm() + temp * 2.0 ** -22 * 8 * w.double().norm() * n ** 0.5


@pytest.mark.parametrize("one_go", [False, True])
@pytest.mark.parametrize("odd", [float("nan"), float("inf")])
@pytest.mark.parametrize("k", [1, 2, 3])
def test_a_teacher_that_is_no_number(k, odd, one_go, monkeypatch):
    """Weights of NaN make their row's loss and gradient NaN, of one token as of several, and no other row's."""
    from dfccl_b200.ops import loss as module
    monkeypatch.setattr(module, "ONE_GO_FROM", 0 if one_go else 1 << 60)
    n, v, d = 40, 300, 64
    x, w, gen = problem(n, v, d, 83)
    t = torch.randint(0, v, (n, 1), generator=gen, device="cuda")
    t = torch.cat([t, t, (t + 1) % v], dim=1)[:, :k]        # (twice the same token, and another)
    teacher = torch.randn(n, k, generator=gen, device="cuda")
    teacher[7, 0] = odd
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    assert module.linear_distillation(a, b, teacher, t, reduction="none").isnan().nonzero()[:, 0].tolist() == [7]
    module.linear_distillation(a, b, teacher, t, reduction="sum").backward()
    assert a.grad.isnan().all(dim=1).nonzero()[:, 0].tolist() == [7] and int(a.grad.isnan().sum()) == d
    assert sorted(b.grad.isnan().all(dim=1).nonzero()[:, 0].tolist()) == sorted(set(t[7].tolist()))


@pytest.mark.parametrize("first", ["targets", "targets, one go", "lists", "lists, one go", "embedding", "gradient of x alone"])
def test_first_calls_of_a_process_are_captured(first):
    """Nothing of this package has run before the capture: what it makes once per device is made beside it."""
    code = f"""
import torch
from dfccl_b200.ops import loss as module
from dfccl_b200.ops.embedding import embedding
from dfccl_b200.ops.gemm import check_kernels
first = {first!r}
module.ONE_GO_FROM = 0 if "one go" in first else 1 << 60
gen = torch.Generator(device="cuda").manual_seed(1)
x, w = torch.randn(50, 64, generator=gen, device="cuda").to(torch.bfloat16), torch.randn(300, 64, generator=gen, device="cuda").to(torch.bfloat16)
t, teacher = torch.randint(0, 300, (50, 3), generator=gen, device="cuda"), torch.randn(50, 3, generator=gen, device="cuda")
leaves = [x.requires_grad_(True)] + ([w] if "alone" in first else [w.requires_grad_(True)])

def step():
    if first == "embedding":
        out = embedding(t, w)
        return (out.detach(),) + torch.autograd.grad(out, [w], torch.ones_like(out))
    out = module.linear_distillation(x, w, teacher, t) if "lists" in first else module.linear_cross_entropy(x, w, t[:, 0])
    return (out.detach(),) + torch.autograd.grad(out, [a for a in leaves if a.requires_grad])

graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
with torch.cuda.graph(graph, stream=side):
    got = step()
graph.replay()
torch.cuda.synchronize()
for a, b in zip(got, step()):
    assert torch.equal(a, b)
assert check_kernels()
"""
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=pathlib.Path(__file__).parents[1])
    assert run.returncode == 0, run.stderr[-2000:]


def test_a_stage_says_what_ran(monkeypatch):
    """Asked for is not run: a head that the loss does not take (its width, its type) leaves the stage's loss to the framework."""
    from dfccl_b200 import native as nv
    from dfccl_b200.models import gpt2
    from dfccl_b200.ops.fused_linear import TpGroup
    (comm,) = nv.Comm.init_loopback(1, torch.cuda.current_device())
    tp = TpGroup(comm, None, torch.device("cuda", torch.cuda.current_device()))
    tokens = torch.randint(0, 300, (2, 129), device="cuda")
    for fused, typed, want in ((False, torch.bfloat16, False), (True, torch.bfloat16, True), (True, torch.float32, False)):
        stage = gpt2.GPT2Stage(gpt2.GPT2Config(n_layer=1, d_model=256, n_head=4, seq_len=128, vocab=300), tp, 0, 1, 2, fused_ends=fused)
        assert not stage.ran_fused_ends
        if typed != torch.bfloat16:
            stage.head = torch.nn.Parameter(stage.head.detach().float())
            monkeypatch.setattr(gpt2, "norm_residual", lambda ln, x: (x, ln(x).float()))
        assert stage(tokens[:, :-1], tokens[:, 1:]).isfinite().item() and stage.ran_fused_ends == want
    comm.destroy()


# more targets than ownSumsKernel takes: sums by sorted tokens, in pieces of the vocabulary; with dw cut into slices (few tiles, long
# contraction) and without (many tiles)
@pytest.mark.parametrize("narrow", [False, True])
@pytest.mark.parametrize("n,v,d,limit", [(6000, 700, 64, 1 << 20), (2500, 9001, 520, 8 << 20), (2100, 20003, 1024, 16 << 20), (4500, 1300, 128, 3 << 20)])
def test_pieces_of_the_vocabulary_by_sorted_targets(n, v, d, limit, narrow, monkeypatch):
    """As test_pieces_of_the_vocabulary, for targets of 64 and of 32 bits and an ignored token of the vocabulary's own."""
    from dfccl_b200.ops import loss as module
    from dfccl_b200.ops.gemm import check_kernels
    monkeypatch.setattr(module, "ONE_GO_FROM", 1 << 60)
    monkeypatch.setenv("DFCCL_LOSS_WORKSPACE_BYTES", str(limit))
    x, w, gen = problem(n, v, d, n + v + d)
    t = (torch.rand(n, generator=gen, device="cuda") ** 3 * v).long().clamp_(max=v - 1)
    ignored = int(t.mode().values)
    keep = t != ignored
    assert n - int(keep.sum()) > 20 and not bool((t[keep] == ignored).any())
    loss, dz = reference(x, w, t[:, None], keep.double()[:, None], 1.0)
    gout = torch.randn(n, generator=gen, device="cuda")
    targets = t.int() if narrow else t
    for want_x, want_w in ((True, True), (True, False), (False, True)):
        a, b = x.clone().requires_grad_(want_x), w.clone().requires_grad_(want_w)
        rows = module.linear_cross_entropy(a, b, targets, ignore_index=ignored, reduction="none")
        check_loss(rows.detach(), loss, x, w, 1.0)
        assert bool((rows.detach()[~keep] == 0).all())
        rows.backward(gout)
        check_gradients((a.grad, b.grad), x, w, dz, gout.double(), 1.0)
        assert not want_x or bool((a.grad[~keep] == 0).all())
        a.grad = b.grad = None
        module.linear_cross_entropy(a, b, targets, ignore_index=ignored, reduction="sum").backward()
        check_gradients((a.grad, b.grad), x, w, dz, torch.ones(n, dtype=torch.float64, device="cuda"), 1.0)
        assert not want_w or bool((b.grad[ignored] != 0).any())          # (the other rows' probabilities of it)
    assert check_kernels()


@pytest.mark.parametrize("limit", [1 << 20, 1 << 30])
@pytest.mark.parametrize("one_go", [False, True])
@pytest.mark.parametrize("n,v,d", [(40, 300, 64), (700, 3001, 136), (3000, 700, 72)])
def test_narrow_targets_and_an_ignored_token_of_the_vocabulary(n, v, d, one_go, limit, monkeypatch):
    """Targets of 32 bits give what those of 64 give, in every piece; a token that is ignored has its share of the others' rows."""
    from dfccl_b200.ops import loss as module
    monkeypatch.setattr(module, "ONE_GO_FROM", 0 if one_go else 1 << 60)
    monkeypatch.setenv("DFCCL_LOSS_WORKSPACE_BYTES", str(limit))
    x, w, gen = problem(n, v, d, 7 * n + v)
    t = torch.randint(0, v, (n,), generator=gen, device="cuda")
    t[::5] = 11
    keep = t != 11
    loss, dz = reference(x, w, t[:, None], keep.double()[:, None], 1.0)
    results = []
    for targets in (t, t.int()):
        a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        value = module.linear_cross_entropy(a, b, targets, ignore_index=11)
        value.backward()
        count = int(keep.sum())
        assert abs(value.item() - loss.sum().item() / count) <= 2 * logit_error(x, w).max().item() + 2 * LN * (1 + loss.abs().max().item())
        check_gradients((a.grad, b.grad), x, w, dz, torch.full((n,), 1.0 / count, dtype=torch.float64, device="cuda"), 1.0, more=2.0 ** -8 * (1 + 2.0 ** -8) if one_go else 0.0)
        assert bool((a.grad[~keep] == 0).all()) and bool((b.grad[11] != 0).any())
        results.append((value.detach(), a.grad, b.grad))
    assert all(torch.equal(p, q) for p, q in zip(*results))


@pytest.mark.parametrize("one_go", [False, True])
@pytest.mark.parametrize("lists", [False, True])
def test_checkpointed_and_moved_to_the_host(lists, one_go, monkeypatch):
    """Inside a checkpoint (the loss runs again in the backward pass), and with what the backward pass needs kept on the host."""
    from torch.utils.checkpoint import checkpoint
    from dfccl_b200.ops import loss as module
    monkeypatch.setattr(module, "ONE_GO_FROM", 0 if one_go else 1 << 60)
    x, w, gen = problem(300, 2001, 128, 91)
    t = torch.randint(0, 2001, (300, 3), generator=gen, device="cuda")
    teacher = torch.randn(300, 3, generator=gen, device="cuda")

    def value(a, b):
        return module.linear_distillation(a, b, teacher, t) if lists else module.linear_cross_entropy(a, b, t[:, 0])

    def gradients(call):
        a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        out = call(a, b)
        out.backward()
        return out.detach(), a.grad, b.grad

    def on_host(a, b):
        with torch.autograd.graph.save_on_cpu():
            return value(a, b)

    want = gradients(value)
    for call in (lambda a, b: checkpoint(value, a, b, use_reentrant=False), lambda a, b: checkpoint(value, a, b, use_reentrant=True), on_host):
        assert all(torch.equal(p, q) for p, q in zip(want, gradients(call)))


@pytest.mark.parametrize("n,v,d,k", [(8192, 128256, 4096, 0), (8192, 128256, 4096, 32), (32768, 50257, 1024, 0), (8192, 50257, 1024, 32), (77, 50257, 768, 0), (100000, 512, 64, 8),
                                     (3, 1000000, 8192, 0), (2000, 30011, 640, 17)])
def test_workspaces_have_the_size_that_is_said(n, v, d, k, monkeypatch):
    """The limit for the probabilities (256 rows or columns at least), 8 bytes an element of the head and 10 of x; beside that 24 bytes and a sixteenth of a row
    an entry, and what does not grow: a few hundred slices of 256 x 256, some stretches of sorted tokens."""
    from dfccl_b200 import native as nv
    L, entries = nv.lib(), n * max(1, k)
    for limit in (1 << 24, 1 << 30):
        monkeypatch.setenv("DFCCL_LOSS_WORKSPACE_BYTES", str(limit))
        least = 256 * 2 * max(v + 64, n)
        most = max(limit, least) * 33 // 32 + 8 * v * d + 10 * n * d + entries * (24 + d // 16) + 2049 * 8 * d + 16 * n + 4 * v + 600 * 2 ** 18 + (1 << 14)
        assert 0 < L.dfcclLinearLossWithGradientsWork(n, v, d, max(1, k), 1, 1) <= most
        assert 0 < L.dfcclLinearLossBackwardWork(n, v, d, k, 1, 1) <= most
