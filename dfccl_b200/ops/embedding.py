"""Embedding of tokens with the gradients of its tables by sorted tokens (``csrc/src/ops/embed.cu``)."""
from __future__ import annotations

import functools
import operator
from typing import Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .. import native as nv
from ..utils.tensors import nccl_dtype, on_device, refuse_tangents, stream_of
from .block import unhooked

TYPES = (torch.bfloat16, torch.float16, torch.float32)


def _index(name: str, t: torch.Tensor) -> None:
    if t.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{name} are int64 or int32, got {t.dtype}")


def _table(name: str, t: torch.Tensor) -> None:
    if t.dim() != 2 or t.shape[0] == 0 or t.shape[1] == 0:
        raise ValueError(f"{name} is [rows, columns], got {tuple(t.shape)}")
    if t.dtype not in TYPES:
        raise ValueError(f"{name} is bf16, fp16 or fp32, got {t.dtype}")
    if t.shape[0] > 2 ** 31 - 16 or t.shape[1] > 2 ** 31 - 4096:
        raise ValueError(f"{name} is {t.shape[0]} x {t.shape[1]}, more than 31 bits count")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """Rows of consecutive elements, however far apart."""
    return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] else t.contiguous()


def _pitch(t: torch.Tensor) -> int:
    """Elements from row to row; of a single row the stride may be anything."""
    return max(t.stride(0), t.shape[1])


def _forward(ids, weight, positions, position_weight, scale):
    n, d = ids.numel(), weight.shape[1]
    out = torch.empty(*ids.shape, d, dtype=weight.dtype, device=weight.device)
    if n == 0:
        return out
    w = _rows(weight)
    if positions is None:
        second = (None, 0, None, 0, 0)
    else:
        p = _rows(position_weight)
        second = (positions.data_ptr(), int(positions.dtype == torch.int64), p.data_ptr(), p.shape[0], _pitch(p))
    with on_device(w.device):
        nv.check(nv.long_entry("dfcclEmbeddingForward")(ids.data_ptr(), int(ids.dtype == torch.int64), n, w.data_ptr(), w.shape[0], _pitch(w), *second, out.data_ptr(),
                                                        d, nccl_dtype(w.dtype), scale, stream_of(w)), "dfcclEmbeddingForward")
    return out


@functools.lru_cache(maxsize=1024)
def _backward_work(n: int, d: int, tables: int) -> int:
    return nv.lib().dfcclEmbeddingBackwardWork(n, d, tables)


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, positions, position_weight, scale, padding):
        ctx.save_for_backward(ids, positions)
        ctx.rows, ctx.prows, ctx.scale, ctx.padding = weight.shape[0], 0 if positions is None else position_weight.shape[0], scale, padding
        ctx.set_materialize_grads(False)
        return _forward(ids, weight, positions, position_weight, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        want_w, want_p = ctx.needs_input_grad[1], ctx.needs_input_grad[3]
        if g is None or not (want_w or want_p):
            return None, None, None, None, None, None
        ids, positions = ctx.saved_tensors
        n, d, device = ids.numel(), g.shape[-1], g.device
        make = torch.empty if n else torch.zeros
        gw = make(ctx.rows, d, dtype=g.dtype, device=device) if want_w else None
        gp = make(ctx.prows, d, dtype=g.dtype, device=device) if want_p else None
        if n:
            g = g.contiguous()
            second = (None, 0, None, 0) if gp is None else (positions.data_ptr(), int(positions.dtype == torch.int64), gp.data_ptr(), ctx.prows)
            with on_device(device):
                work = torch.empty(_backward_work(n, d, want_w + want_p), dtype=torch.uint8, device=device)
                nv.check(nv.long_entry("dfcclEmbeddingBackward")(g.data_ptr(), n, d, nccl_dtype(g.dtype), ids.data_ptr(), int(ids.dtype == torch.int64), ctx.padding,
                                                                 ctx.scale, None if gw is None else gw.data_ptr(), ctx.rows, *second, work.data_ptr(), stream_of(g)),
                         "dfcclEmbeddingBackward")
        return None, gw, None, gp, None, None


def lookup_supported(tokens: nn.Module, positions: nn.Module) -> bool:
    """True if ``embedding`` of the two modules' tables is what calling them and adding their results gives: modules that look up and
    do nothing else (no row without a gradient, renormalised, scaled by its count or of a sparse gradient), tables of one kind."""
    a, b = tokens, positions
    return (all(unhooked(m, nn.Embedding) and m.padding_idx is None and m.max_norm is None and not m.scale_grad_by_freq and not m.sparse for m in (a, b))
            and a.weight.dtype == b.weight.dtype and a.weight.dtype in TYPES and a.weight.device == b.weight.device
            and a.weight.shape[1] == b.weight.shape[1])


def embedding(ids: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0, positions: Optional[torch.Tensor] = None,
              position_weight: Optional[torch.Tensor] = None, padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * weight[ids] + position_weight[positions]``, computed in fp32 and rounded once; [*ids.shape, columns].

    ``weight`` and ``position_weight`` (both or neither of the position arguments) are bf16, fp16 or fp32 of one type, ``ids``
    and ``positions`` int64 or int32 of one shape.  The gradients of both tables are dense; each row of them is the fp32 sum over
    its tokens (in their order within stretches of 16 to 128, whose sums are added up behind that), rounded once, the same in every run.  Tokens ``padding_idx`` give ``weight`` none.  There is no check of the
    ids' values on the host: a token outside its table gives a row of NaN and no gradient of that table."""
    _index("ids", ids)
    _table("weight", weight)
    if (positions is None) != (position_weight is None):
        raise ValueError("positions and position_weight belong together")
    device = weight.device
    here = device.type == "cuda" and ids.device == device
    if positions is not None:
        _index("positions", positions)
        _table("position_weight", position_weight)
        if positions.shape != ids.shape:
            raise ValueError(f"positions of {tuple(positions.shape)} for ids of {tuple(ids.shape)}")
        if position_weight.shape[1] != weight.shape[1] or position_weight.dtype != weight.dtype:
            raise ValueError(f"position_weight of {tuple(position_weight.shape)} {position_weight.dtype} beside weight of {tuple(weight.shape)} {weight.dtype}")
        here = here and positions.device == device and position_weight.device == device
        positions = positions.contiguous()
    padding = -1 if padding_idx is None else operator.index(padding_idx)
    if padding_idx is not None and not 0 <= padding < weight.shape[0]:
        raise ValueError(f"padding_idx {padding_idx} outside a table of {weight.shape[0]} rows")
    if ids.numel() > 2 ** 31 - 4096:
        raise ValueError(f"{ids.numel()} tokens in one call, more than 31 bits count")
    refuse_tangents(weight, position_weight)
    if not here:
        raise ValueError("the embedding runs on tensors of one GPU")
    ids, scale = ids.contiguous(), float(scale)
    if torch.is_grad_enabled() and (weight.requires_grad or (position_weight is not None and position_weight.requires_grad)):
        return _EmbeddingFn.apply(ids, weight, positions, position_weight, scale, padding)
    return _forward(ids, weight, positions, position_weight, scale)
