"""Losses of a language model's head from the head's inputs and weights, without keeping the logits (``csrc/src/ops/loss.cu``,
``csrc/src/gemm/tcgen05_vocab.cu``): cross entropy with a target per row, distillation from a teacher's top logits."""
from __future__ import annotations

import functools
import operator

import torch
from torch.autograd.function import once_differentiable

from .. import native as nv
from ..utils.tensors import nccl_dtype, on_device, refuse_tangents, stream_of
from .block import packed

REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}
MAX_LIST = 256                       # entries of a teacher's list
# Rows x vocabulary (counted as SMALL_VOCABULARY at least beside targets) above which a reduced loss makes its gradients with the loss.  GPU time in us,
# logits computed twice / once: targets 512 x 50257 x 64 75 / 79, 1024 x 50257 x 64 115 / 108, x 256 140 / 132, 2048 x 2000 x 256 59 / 62, 3000 x 2000 x 256
# 75 / 68, 3000 x 500 x 64 62 / 54.  A head whose way from memory takes longer than what one go has more to launch: targets 64 x 50257 x 512 97 / 102, x 768
# 110 / 108, x 1024 134 / 132; 512 x 50257 x 1024 220 / 203; 64 x 131072 x 1024 279 / 251, x 4096 996 / 840; lists of 8 64 x 50257 x 64 74 / 80, x 768
# 137 / 133, x 1024 164 / 158, 64 x 32000 x 4096 408 / 383.  Lists of more than 2048 entries together, which both ways sort: lists of 8 256 x 2000 x 64 55 / 62,
# 300 68 / 64, 2048 80 / 72; 256 x 8000 x 256 68 / 74, of 64 100 / 98; of 32 8192 x 8000 x 256 381 / 299, 256 x 32000 x 4096 502 / 512, 2048 1622 / 1294; of 17
# 1777 x 30011 x 640 287 / 242, of 128 496 / 404; of 256 4096 x 50257 x 1024 2238 / 1755.
ONE_GO_FROM = 2 ** 25
SMALL_VOCABULARY = 14000            # of 2400 rows
LARGE_HEAD = 0.8                     # of 2 ** 25 / 0.8 elements
LIST_SHARE = 2 ** 14                 # an entry of a list: of 2048 entries
MOST_ROWS = 2 ** 31 - 1 - 2 ** 20     # 31 bits, less what loops over pieces of them go past their end
MOST_ENTRIES = 2 ** 31 - 4097        # of all lists together, as their sorting counts them


def linear_loss_supported(x: torch.Tensor, weight: torch.Tensor) -> bool:
    """True if the losses of this module take ``x`` [..., d] and ``weight`` [vocabulary, d]."""
    return (x.is_cuda and x.device == weight.device and x.dtype == weight.dtype == torch.bfloat16 and x.dim() >= 1 and weight.dim() == 2
            and weight.shape[0] > 0 and x.shape[-1] == weight.shape[1] and weight.shape[1] > 0 and weight.shape[1] % 8 == 0)


def _check(x: torch.Tensor, weight: torch.Tensor, index: torch.Tensor, name: str, reduction: str) -> None:
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction is one of {', '.join(REDUCTIONS)}, got {reduction!r}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x [..., d] and weight [vocabulary, d], got {tuple(x.shape)} and {tuple(weight.shape)}")
    if x.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise ValueError(f"x and weight are bf16, got {x.dtype} and {weight.dtype}")
    v, d = weight.shape
    if d == 0 or d % 8 or v == 0:
        raise ValueError(f"the width is a multiple of 8 and the vocabulary not empty, got {v} x {d}")
    if index.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{name} are int64 or int32, got {index.dtype}")
    if max(x.numel() // d, v, d) > MOST_ROWS:
        raise ValueError(f"at most {MOST_ROWS} rows, entries of the vocabulary and columns, got {x.numel() // d} x {v} x {d}")
    refuse_tangents(x, weight)


def _on_one_gpu(device: torch.device, *tensors: torch.Tensor) -> None:
    if device.type != "cuda" or any(t.device != device for t in tensors):
        raise ValueError("the losses run on tensors of one GPU")


@functools.lru_cache(maxsize=1024)
def _forward_work(n: int, v: int, k: int) -> int:
    return nv.lib().dfcclLinearLossForwardWork(n, v, k)


class _Rows:
    """What the rows are compared with, as the C interface takes it: a target each, or lists of ``k`` entries (of ``entries`` in
    all: their tokens, behind them their weights, behind those the rows' states, 32 bits each)."""
    __slots__ = ("targets", "ignore", "lists", "entries", "k", "temperature")

    def __init__(self, targets, ignore, lists, entries, k, temperature):
        self.targets, self.ignore, self.lists, self.entries, self.k, self.temperature = targets, ignore, lists, entries, k, temperature

    def tensor(self):
        return self.targets if self.lists is None else self.lists

    def args(self):
        if self.lists is None:
            return self.targets.data_ptr(), int(self.targets.dtype == torch.int64), self.ignore, None, None, None, 1, 1.0
        at = self.lists.data_ptr()
        return None, 0, 0, at, at + 4 * self.entries, at + 8 * self.entries, self.k, self.temperature


def _forward(x, weight, rows, reduction, keep):
    """(loss, x and weight as the kernels read them, what the backward pass needs of the sums where ``keep`` is set)."""
    v, d = weight.shape
    n, device = x.numel() // d, x.device
    xp, wp = packed(x), packed(weight)
    # log2 of the sums, the number of rows that count, what is left of the weights; where nobody wants them, behind the workspace
    words, behind = n + 1 + n * rows.k, 0 if keep or not n else _forward_work(n, v, rows.k) // 4
    kept = torch.empty(behind + words, dtype=torch.float32, device=device)
    loss = kept.new_empty(() if reduction else x.shape[:-1])
    if n:
        at, out = kept.data_ptr() + 4 * behind, loss.data_ptr()
        with on_device(device):
            work = kept if behind else torch.empty(_forward_work(n, v, rows.k), dtype=torch.uint8, device=device)
            nv.check(nv.long_entry("dfcclLinearLossForward")(xp.data_ptr(), wp.data_ptr(), n, v, d, *rows.args(), reduction, work.data_ptr(), at, at + 4 * (n + 1),
                                                             None if reduction else out, out if reduction else None, at + 4 * n if reduction else None,
                                                             stream_of(x)), "dfcclLinearLossForward")
    elif reduction:
        loss.zero_()
    return loss, xp, wp, kept


def _forward_with_gradients(x, weight, rows, reduction, want_x, want_w):
    """What ``_forward`` returns, and the gradients of x and weight for a gradient of 1 of the loss."""
    v, d = weight.shape
    n, device = x.numel() // d, x.device
    xp, wp = packed(x), packed(weight)
    kept = torch.empty(n + 1 + n * rows.k, dtype=torch.float32, device=device)
    loss = kept.new_empty(())
    dx = torch.empty_like(xp) if want_x else None
    dw = torch.empty_like(wp) if want_w else None
    at = kept.data_ptr()
    with on_device(device):
        size = nv.lib().dfcclLinearLossWithGradientsWork(n, v, d, rows.k, want_x, want_w)
        work = torch.empty(size, dtype=torch.uint8, device=device)
        nv.check(nv.long_entry("dfcclLinearLossWithGradients")(xp.data_ptr(), wp.data_ptr(), n, v, d, *rows.args(), reduction, work.data_ptr(), size, at, at + 4 * (n + 1),
                                                               loss.data_ptr(), at + 4 * n, dx.data_ptr() if want_x else None,
                                                               dw.data_ptr() if want_w else None, stream_of(x)), "dfcclLinearLossWithGradients")
    return loss, xp, wp, kept, (dx, dw)


def _scaled(grads, g):
    """The gradients times that of the loss, in place: nothing else holds them, and whatever runs this again makes them anew."""
    dx, dw = grads
    with on_device(g.device):
        nv.check(nv.entry("dfcclScaleResults")(None if dx is None else dx.data_ptr(), 0 if dx is None else dx.numel(), None if dw is None else dw.data_ptr(),
                                               0 if dw is None else dw.numel(), g.data_ptr(), stream_of(g)), "dfcclScaleResults")
    return dx, dw, None, None


class _LinearLossFn(torch.autograd.Function):
    """A reduced loss of some size makes its gradients with the loss, which saves computing the logits a second time: the first
    backward pass scales them.  Another pass over the same graph, one captured into a CUDA graph that has not captured the loss
    (its replays would scale what they have scaled before), and every other loss, computes the logits again."""

    @staticmethod
    def forward(ctx, x, weight, rows, reduction):
        want_x, want_w = ctx.needs_input_grad[:2]
        ctx.grads = None
        n, v = x.numel() // weight.shape[1], weight.shape[0]
        least = n * max(v, SMALL_VOCABULARY) if rows.lists is None else max(n * v, rows.entries * LIST_SHARE)
        one_go = max(least, weight.numel() * LARGE_HEAD) > ONE_GO_FROM and rows.entries <= MOST_ENTRIES
        if n and reduction and (want_x or want_w) and one_go:
            loss, xp, wp, kept, ctx.grads = _forward_with_gradients(x, weight, rows, reduction, want_x, want_w)
            ctx.capture = nv.lib().dfcclCaptureId(stream_of(x))
        else:
            loss, xp, wp, kept = _forward(x, weight, rows, reduction, True)
        ctx.save_for_backward(xp, wp, kept, rows.tensor())
        ctx.rows, ctx.mean = rows, reduction == 1
        ctx.set_materialize_grads(False)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        want_x, want_w = ctx.needs_input_grad[:2]
        if g is None or not (want_x or want_w):
            return None, None, None, None
        x, w, kept = ctx.saved_tensors[:3]                  # (asking for them notices a change in place, of the targets too)
        grads, ctx.grads = ctx.grads, None
        if grads is not None and ctx.capture == nv.lib().dfcclCaptureId(stream_of(x)):
            return _scaled(grads, g)
        (v, d), device = w.shape, x.device
        n = x.numel() // d
        if n == 0:
            return torch.zeros_like(x) if want_x else None, torch.zeros_like(w) if want_w else None, None, None
        g = g.reshape(-1) if g.dim() else g
        dx = torch.empty_like(x) if want_x else None
        dw = torch.empty_like(w) if want_w else None
        with on_device(device):
            size = nv.lib().dfcclLinearLossBackwardWork(n, v, d, 0 if ctx.rows.lists is None else ctx.rows.k, want_x, want_w)
            work = torch.empty(size, dtype=torch.uint8, device=device)
            at = kept.data_ptr()
            nv.check(nv.long_entry("dfcclLinearLossBackward")(x.data_ptr(), w.data_ptr(), n, v, d, *ctx.rows.args(), at, at + 4 * (n + 1), g.data_ptr(),
                                                              g.stride(0) if g.dim() else 0, at + 4 * n if ctx.mean else None, dx.data_ptr() if want_x else None,
                                                              dw.data_ptr() if want_w else None, work.data_ptr(), size, stream_of(x)), "dfcclLinearLossBackward")
        return dx, dw, None, None


def _loss(x, weight, rows, reduction):
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        return _LinearLossFn.apply(x, weight, rows, REDUCTIONS[reduction])
    return _forward(x, weight, rows, REDUCTIONS[reduction], False)[0]


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """Softmax cross entropy of the logits ``x @ weight.T`` with ``targets``, in fp32; the logits are not stored.

    ``x`` [..., d] and ``weight`` [vocabulary, d] are bf16, d a multiple of 8; ``targets`` [...] int64 or int32.  Rows of target
    ``ignore_index`` have no loss and give no gradient, whatever ``x`` holds there; ``"mean"`` is over the other rows, and 0 where
    there is none.  Logits (up to 2**30 in size) and sums are fp32; the probabilities are rounded to bf16 on their way into the products that make the
    gradients of ``x`` and ``weight``, what the targets add to them is not.  They exist for as many columns or rows at a time as
    ``DFCCL_LOSS_WORKSPACE_BYTES`` (1 GiB) hold, 256 at least; beside them sums in fp32 take up to 8 bytes an element of ``weight`` and 10 an
    element of ``x``, and up to 0.2 GB (8192 rows over 128256 x 4096: 3.4 GB in all).

    Large reduced losses make their gradients with the loss and keep them until the first backward pass, which multiplies them by the
    gradient of the loss where that is not 1.  If it is no power of two, they are rounded to bf16 a second time there (1.7e-3 off in the
    2-norm becomes 2.3e-3); small losses take it into the first rounding.  A row whose loss is above 41 makes such a pass half as long again.

    There is no check of the targets' values on the host: one outside the vocabulary makes its row's loss and gradients NaN."""
    _check(x, weight, targets, "targets", reduction)
    if targets.shape != x.shape[:-1]:
        raise ValueError(f"targets of {tuple(targets.shape)} for x of {tuple(x.shape)}")
    ignore_index = operator.index(ignore_index)
    if not -2 ** 63 <= ignore_index < 2 ** 63:
        raise ValueError(f"ignore_index {ignore_index} is no token of 64 bits")
    _on_one_gpu(x.device, weight, targets)
    return _loss(x, weight, _Rows(targets.contiguous(), ignore_index, None, targets.numel(), 1, 1.0), reduction)


def linear_distillation(x: torch.Tensor, weight: torch.Tensor, teacher_logits: torch.Tensor, teacher_tokens: torch.Tensor, *, temperature: float = 1.0,
                        reduction: str = "mean") -> torch.Tensor:
    """Divergence of the student's distribution from the teacher's top logits, ``T^2 sum_k q_k (ln q_k - ln p_k)`` per row: q is the
    softmax of ``teacher_logits / T`` over the row's entries, p that of ``x @ weight.T / T`` over the whole vocabulary, read at
    ``teacher_tokens``.

    ``x`` and ``weight`` as in ``linear_cross_entropy``, T 2**-20 to 2**20 (a loss is exact to T^2 times a rounding or two of fp32); ``teacher_logits`` [..., k] fp32, bf16 or fp16 and ``teacher_tokens`` [..., k]
    int64 or int32, k up to 256 in any order.  Entries of token -1 or of logit -inf are left out; a row without any has no loss and
    gives no gradient.  A token that stands in a row twice counts as two entries.  ``"mean"`` is over the rows with entries, 0 where
    there is none.  No gradient (and no tangent) reaches the teacher.  Any other token outside the vocabulary makes its row NaN."""
    _check(x, weight, teacher_tokens, "teacher_tokens", reduction)
    if teacher_tokens.dim() != x.dim() or teacher_tokens.shape[:-1] != x.shape[:-1] or teacher_logits.shape != teacher_tokens.shape:
        raise ValueError(f"teacher_logits of {tuple(teacher_logits.shape)} and teacher_tokens of {tuple(teacher_tokens.shape)} for x of {tuple(x.shape)}")
    if teacher_logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError(f"teacher_logits are fp32, bf16 or fp16, got {teacher_logits.dtype}")
    k = teacher_tokens.shape[-1]
    if not 1 <= k <= MAX_LIST:
        raise ValueError(f"lists of 1 to {MAX_LIST} entries, got {k}")
    if not 2.0 ** -20 <= temperature <= 2.0 ** 20:
        raise ValueError(f"the temperature is 2**-20 to 2**20, got {temperature}")
    device, temperature = x.device, float(temperature)
    _on_one_gpu(device, weight, teacher_logits, teacher_tokens)
    n, v = teacher_tokens.numel() // k, weight.shape[0]
    lists = torch.empty(2 * n * k + n, dtype=torch.int32, device=device)
    rows = _Rows(None, 0, lists, n * k, k, temperature)
    logits, listed = teacher_logits.detach().contiguous(), teacher_tokens.contiguous()
    if n:
        with on_device(device):
            nv.check(nv.long_entry("dfcclTeacherRows")(logits.data_ptr(), nccl_dtype(logits.dtype), listed.data_ptr(), int(listed.dtype == torch.int64), n, k, v,
                                               temperature, *rows.args()[3:6], stream_of(x)), "dfcclTeacherRows")
    return _loss(x, weight, rows, reduction)
