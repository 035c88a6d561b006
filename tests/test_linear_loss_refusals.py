"""What the embedding and the losses over a vocabulary refuse, before anything reaches a GPU."""
import ctypes as C

import pytest
import torch

BF = torch.bfloat16


def x(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def i(*shape, dtype=torch.int64):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("args,kw,what", [
    ((x(4, 16), x(9, 16), i(4)), {"reduction": "average"}, "reduction"),
    ((x(4, 16), x(9, 24), i(4)), {}, "x \\[..., d\\]"),
    ((x(4, 16), x(16), i(4)), {}, "x \\[..., d\\]"),
    ((x(4, 16, dtype=torch.float32), x(9, 16, dtype=torch.float32), i(4)), {}, "bf16"),
    ((x(4, 16), x(9, 16, dtype=torch.float16), i(4)), {}, "bf16"),
    ((x(4, 12), x(9, 12), i(4)), {}, "multiple of 8"),
    ((x(4, 0), x(9, 0), i(4)), {}, "multiple of 8"),
    ((x(4, 16), x(0, 16), i(4)), {}, "not empty"),
    ((x(4, 16), x(9, 16), i(4, dtype=torch.int16)), {}, "int64 or int32"),
    ((x(4, 16), x(9, 16), i(5)), {}, "targets of"),
    ((x(4, 16), x(9, 16), i(4, 1)), {}, "targets of"),
    ((x(4, 16), x(9, 16), i(4)), {}, "GPU")])
def test_cross_entropy_refuses(args, kw, what):
    from dfccl_b200.ops.loss import linear_cross_entropy
    with pytest.raises(ValueError, match=what):
        linear_cross_entropy(*args, **kw)


@pytest.mark.parametrize("args,kw,what", [
    ((x(4, 16), x(9, 16), x(4, 3), i(4, 2)), {}, "teacher_logits of"),
    ((x(4, 16), x(9, 16), x(4), i(4)), {}, "teacher_logits of"),
    ((x(4, 16), x(9, 16), x(5, 2), i(5, 2)), {}, "teacher_logits of"),
    ((x(4, 16), x(9, 16), i(4, 2), i(4, 2)), {}, "fp32, bf16 or fp16"),
    ((x(4, 16), x(9, 16), x(4, 2), x(4, 2)), {}, "int64 or int32"),
    ((x(4, 16), x(9, 16), x(4, 0), i(4, 0)), {}, "1 to 256"),
    ((x(4, 16), x(9, 16), x(4, 257), i(4, 257)), {}, "1 to 256"),
    ((x(4, 16), x(9, 16), x(4, 2), i(4, 2)), {"temperature": 0.0}, "temperature"),
    ((x(4, 16), x(9, 16), x(4, 2), i(4, 2)), {"temperature": float("nan")}, "temperature"),
    ((x(4, 16), x(9, 16), x(4, 2), i(4, 2)), {"temperature": float("inf")}, "temperature"),
    ((x(4, 16), x(9, 16), x(4, 2), i(4, 2)), {}, "GPU")])
def test_distillation_refuses(args, kw, what):
    from dfccl_b200.ops.loss import linear_distillation
    with pytest.raises(ValueError, match=what):
        linear_distillation(*args, **kw)


@pytest.mark.parametrize("args,kw,what", [
    ((i(4, dtype=torch.uint8), x(9, 16)), {}, "int64 or int32"),
    ((i(4), x(16)), {}, "weight is"),
    ((i(4), x(0, 16)), {}, "weight is"),
    ((i(4), x(9, 0)), {}, "weight is"),
    ((i(4), x(9, 16, dtype=torch.float64)), {}, "bf16, fp16 or fp32"),
    ((i(4), x(9, 16)), {"positions": i(4)}, "belong together"),
    ((i(4), x(9, 16)), {"position_weight": x(9, 16)}, "belong together"),
    ((i(4), x(9, 16)), {"positions": i(5), "position_weight": x(9, 16)}, "positions of"),
    ((i(4), x(9, 16)), {"positions": x(4), "position_weight": x(9, 16)}, "int64 or int32"),
    ((i(4), x(9, 16)), {"positions": i(4), "position_weight": x(9, 24)}, "beside weight"),
    ((i(4), x(9, 16)), {"positions": i(4), "position_weight": x(9, 16, dtype=torch.float32)}, "beside weight"),
    ((i(4), x(9, 16)), {"padding_idx": 9}, "padding_idx"),
    ((i(4), x(9, 16)), {"padding_idx": -1}, "padding_idx"),
    ((i(4), x(9, 16)), {}, "GPU")])
def test_embedding_refuses(args, kw, what):
    from dfccl_b200.ops.embedding import embedding
    with pytest.raises(ValueError, match=what):
        embedding(*args, **kw)


def test_entries_refuse(native):
    """The C entry points answer with a status: no null pointers, no odd widths, no lists beyond the limit, no misaligned operands."""
    L, bad, p, q = native.lib(), native.INVALID_ARGUMENT, 4096, 4100
    assert L.dfcclLinearLossMaxList() == 256
    ok = [p, p, 4, 9, 16, p, 1, -100, None, None, None, 1, 1.0, 0, p, p, p, p, None, None, None]
    for at, value in ((0, None), (1, q), (2, 0), (3, 0), (4, 12), (5, None), (11, 0), (11, 2), (12, 0.0), (13, 3), (13, 1), (14, None), (15, None), (16, None), (17, None)):
        args = list(ok)
        args[at] = value
        assert L.dfcclLinearLossForward(*args) == bad, (at, value)
    lists = ok[:5] + [None, 0, 0, p, p, p, 8] + ok[12:]
    for at, value in ((8, None), (9, None), (10, None), (11, 257)):
        args = list(lists)
        args[at] = value
        assert L.dfcclLinearLossForward(*args) == bad, (at, value)
    ok = [p, p, 4, 9, 16, p, 1, -100, None, None, None, 1, 1.0, p, p, p, 0, None, p, p, p, 1 << 30, None]
    for at, value in ((0, None), (1, q), (2, -1), (4, 4), (5, None), (11, 300), (12, -1.0), (13, None), (14, None), (15, None), (16, -1), (18, q), (19, q), (20, None), (21, 16)):
        args = list(ok)
        args[at] = value
        assert L.dfcclLinearLossBackward(*args) == bad, (at, value)
    args = list(ok)
    args[18] = args[19] = None
    assert L.dfcclLinearLossBackward(*args) == bad
    assert L.dfcclLinearLossForwardWork(4, 9, 0) == 0 and L.dfcclLinearLossBackwardWork(4, 9, 16, 0, 0, 0) == 0 and L.dfcclLinearLossBackwardWork(4, 9, 16, 257, 1, 1) == 0
    ok = [p, p, 4, 9, 16, p, 1, -100, None, None, None, 1, 1.0, 1, p, 1 << 30, p, p, p, p, p, p, None]
    for at, value in ((0, None), (1, q), (2, 0), (4, 12), (5, None), (11, 2), (12, 0.0), (13, 0), (13, 3), (14, None), (15, 16), (16, None), (17, None), (18, None), (19, None),
                      (20, q), (21, q)):
        args = list(ok)
        args[at] = value
        assert L.dfcclLinearLossWithGradients(*args) == bad, (at, value)
    assert L.dfcclLinearLossWithGradientsWork(4, 9, 16, 1, 0, 0) == 0 and L.dfcclLinearLossWithGradientsWork(4, 9, 16, 1, 1, 0) > 0
    assert L.dfcclLinearLossWithGradientsWork(2 ** 24, 9, 16, 256, 1, 1) == 0
    for args in ((p, 12, None, 0, p, None), (q, 16, None, 0, p, None), (None, 16, None, 0, p, None), (None, 0, None, 0, p, None), (p, 16, p, 16, None, None)):
        assert L.dfcclScaleResults(*args) == bad
    assert L.dfcclTeacherRows(p, native.INT32, p, 1, 4, 2, 9, 1.0, p, p, p, None) == bad and L.dfcclTeacherRows(p, native.FLOAT32, p, 1, 4, 257, 9, 1.0, p, p, p, None) == bad
    ok = [p, 1, 4, p, 9, 16, None, 0, None, 0, 0, p, 16, native.BFLOAT16, 1.0, None]
    for at, value in ((0, None), (2, 0), (3, None), (4, 0), (5, 8), (6, p), (11, None), (12, 0), (13, native.FLOAT64)):
        args = list(ok)
        args[at] = value
        assert L.dfcclEmbeddingForward(*args) == bad, (at, value)
    ok = [p, 4, 16, native.BFLOAT16, p, 1, -1, 1.0, p, 9, None, 0, None, 0, p, None]
    for at, value in ((0, None), (1, 0), (2, 0), (3, native.INT64), (4, None), (8, None), (8, q), (9, 0), (9, 2 ** 31), (12, p), (14, None)):
        args = list(ok)
        args[at] = value
        assert L.dfcclEmbeddingBackward(*args) == bad, (at, value)
    assert L.dfcclEmbeddingBackwardWork(4, 16, 3) == 0 and L.dfcclEmbeddingBackwardWork(4, 16, 2) > 0
    assert isinstance(L.dfcclLinearLossBackwardWork(1000, 50257, 1024, 0, 1, 1), int) and C.sizeof(C.c_size_t) == 8


def test_long_entries(native):
    """Entry points of many arguments: integers, None and a float wherever it stands, as ctypes passes them; nothing else."""
    import numpy as np
    f, g = native.long_entry("dfcclEmbeddingBackward"), native.lib().dfcclEmbeddingBackward
    assert native.long_entry("dfcclEmbeddingBackward") is f
    ok = [4096, 4, 16, native.BFLOAT16, 4096, 1, -1, 1.0, 4100, 9, None, 0, None, 0, 4096, None]          # (misaligned: refused)
    assert f(*ok) == g(*ok) == native.INVALID_ARGUMENT
    if native._hostcall() is None:
        return
    call = native._hostcall_module.call_long
    libc = C.CDLL(None)
    assert call(C.cast(libc.abs, C.c_void_p).value, -7) == 7
    assert call(C.cast(libc.lrintf, C.c_void_p).value, 41.6) == 42 and call(C.cast(libc.ilogbf, C.c_void_p).value, None, 8.5, 3) == 3
    text = [C.create_string_buffer(t) for t in (b"abcd", b"abxy")]
    where = C.cast(libc.strncmp, C.c_void_p).value
    assert call(where, *(C.addressof(t) for t in text), np.int64(2)) == 0 and call(where, *(C.addressof(t) for t in text), 3) < 0
    for bad in ((1.5,), (None,), (1, 1.0, 2.0), (1, "x"), tuple([1] * 26), ()):
        with pytest.raises(TypeError):
            call(*bad)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("which", range(6))
def test_tangents_are_refused(which, grad):
    """A forward-mode derivative is not computed, and not dropped either: of every operand that has a derivative, in and out of no_grad."""
    import torch.autograd.forward_ad as fw
    from dfccl_b200.ops.embedding import embedding
    from dfccl_b200.ops.loss import linear_cross_entropy, linear_distillation
    with fw.dual_level(), torch.set_grad_enabled(grad):
        a, w = x(4, 16), x(9, 16)
        with_tangent = fw.make_dual(x(4, 16) if which in (0, 2) else x(9, 16), torch.ones(4 if which in (0, 2) else 9, 16, dtype=BF))
        call = [lambda t: linear_cross_entropy(t, w, i(4)), lambda t: linear_cross_entropy(a, t, i(4)),
                lambda t: linear_distillation(t, w, x(4, 2), i(4, 2)), lambda t: linear_distillation(a, t, x(4, 2), i(4, 2)),
                lambda t: embedding(i(4), t), lambda t: embedding(i(4), w, positions=i(4), position_weight=t)][which]
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(with_tangent)
        with pytest.raises(ValueError, match="GPU"):
            call(fw.unpack_dual(with_tangent).primal)


def test_sizes_at_the_end_of_31_bits(native):
    """Loops over pieces of rows or columns count past their end by up to a piece: sizes whose count would not fit are refused."""
    from dfccl_b200.ops.embedding import embedding
    from dfccl_b200.ops.loss import MOST_ROWS, linear_cross_entropy, linear_distillation
    L, top = native.lib(), 2 ** 31
    assert top - 2 ** 21 < MOST_ROWS < top - 742000
    for n, v, d in ((MOST_ROWS + 1, 9, 8), (4, MOST_ROWS + 1, 8), (top - 4096, 9, 8), (100, top - 4096, 8), (4, 9, top - 8)):
        assert L.dfcclLinearLossWithGradientsWork(n, v, d, 1, 1, 1) == 0 and L.dfcclLinearLossBackwardWork(n, v, d, 0, 1, 1) == 0
        assert d > 8 or L.dfcclLinearLossForwardWork(n, v, 1) == 0
        rows, head = x(1, 1).expand(n, d), x(1, 1).expand(v, d)
        with pytest.raises(ValueError, match="at most"):
            linear_cross_entropy(rows, head, i(1).expand(n))
        with pytest.raises(ValueError, match="at most"):
            linear_distillation(rows, head, x(1, 1).expand(n, 2), i(1, 1).expand(n, 2))
    assert L.dfcclLinearLossForwardWork(MOST_ROWS, 9, 1) > 0
    assert L.dfcclEmbeddingBackwardWork(top - 4095, 8, 1) == 0 and L.dfcclEmbeddingBackwardWork(top - 4096, 8, 1) > 0
    p = 4096
    assert L.dfcclEmbeddingForward(p, 1, top - 1, p, 9, 16, None, 0, None, 0, 0, p, 16, native.BFLOAT16, 1.0, None) == native.INVALID_ARGUMENT
    assert L.dfcclEmbeddingBackward(p, top - 1, 16, native.BFLOAT16, p, 1, -1, 1.0, p, 9, None, 0, None, 0, p, None) == native.INVALID_ARGUMENT
    with pytest.raises(ValueError, match="31 bits"):
        embedding(i(4), x(1, 1).expand(9, top + 8))
    with pytest.raises(ValueError, match="31 bits"):
        embedding(i(1).expand(top - 4095), x(9, 16))


def test_entries_refuse_misaligned_workspaces(native):
    """A workspace is accessed 32 bytes at a time: one that starts elsewhere is an invalid argument, not a fault."""
    L, bad, p = native.lib(), native.INVALID_ARGUMENT, 4096
    entries = [(L.dfcclLinearLossForward, [p, p, 4, 9, 16, p, 1, -100, None, None, None, 1, 1.0, 0, p, p, p, p, None, None, None], 14),
               (L.dfcclLinearLossBackward, [p, p, 4, 9, 16, p, 1, -100, None, None, None, 1, 1.0, p, p, p, 0, None, p, p, p, 1 << 30, None], 20),
               (L.dfcclLinearLossWithGradients, [p, p, 4, 9, 16, p, 1, -100, None, None, None, 1, 1.0, 1, p, 1 << 30, p, p, p, p, p, p, None], 14),
               (L.dfcclEmbeddingBackward, [p, 4, 16, native.BFLOAT16, p, 1, -1, 1.0, p, 9, None, 0, None, 0, p, None], 14)]
    for entry, args, work in entries:
        for off in (4, 8, 16, 31):
            assert entry(*args[:work], p + off, *args[work + 1:]) == bad, (entry, off)


def test_what_is_no_token():
    """An ignored token or a padding token is a whole number that the kernels' 64 bits hold; None, a float or more bits are not read as token 0."""
    import numpy as np
    from dfccl_b200.ops.embedding import embedding
    from dfccl_b200.ops.loss import linear_cross_entropy
    for bad in (None, 0.0, -100.0, "0"):
        with pytest.raises(TypeError):
            linear_cross_entropy(x(4, 16), x(9, 16), i(4), ignore_index=bad)
    for bad in (2 ** 63, 2 ** 64, -2 ** 63 - 1):
        with pytest.raises(ValueError, match="64 bits"):
            linear_cross_entropy(x(4, 16), x(9, 16), i(4), ignore_index=bad)
    for good in (-2 ** 63, 2 ** 63 - 1, np.int32(3), torch.tensor(5)):
        with pytest.raises(ValueError, match="GPU"):
            linear_cross_entropy(x(4, 16), x(9, 16), i(4), ignore_index=good)
    for bad in (2.0, 2.5, "0"):
        with pytest.raises(TypeError):
            embedding(i(4), x(9, 16), padding_idx=bad)
    for good in (np.int64(3), 8):
        with pytest.raises(ValueError, match="GPU"):
            embedding(i(4), x(9, 16), padding_idx=good)


@pytest.mark.parametrize("temperature", [1e-45, 1e-25, 1e-7, 2.0 ** -20 * 0.99, 2.0 ** 20 * 1.01, 1e20, 1e39])
def test_temperatures_out_of_range(native, temperature):
    """Whose square, inverse or exponents fp32 does not hold: an error, not NaN."""
    from dfccl_b200.ops.loss import linear_distillation
    with pytest.raises(ValueError, match="temperature"):
        linear_distillation(x(4, 16), x(9, 16), x(4, 2), i(4, 2), temperature=temperature)
    for ok in (2.0 ** -20, 2.0 ** 20):
        with pytest.raises(ValueError, match="GPU"):
            linear_distillation(x(4, 16), x(9, 16), x(4, 2), i(4, 2), temperature=ok)
    L, p = native.lib(), 4096
    assert L.dfcclTeacherRows(p, native.FLOAT32, p, 1, 4, 2, 9, temperature, p, p, p, None) == native.INVALID_ARGUMENT
    assert L.dfcclLinearLossForward(p, p, 4, 9, 16, None, 0, 0, p, p, p, 2, temperature, 0, p, p, p, p, None, None, None) == native.INVALID_ARGUMENT
