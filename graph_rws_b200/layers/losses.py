"""Losses over the class axis on the library's kernels (csrc/linear_ce.cu, csrc/distill.cu): softmax cross entropy of a
linear classifier that never keeps its scores, and distillation from a teacher's best scores.  The reference's steps take
F.cross_entropy of the last layer's output (helper/engine.py:66-75)."""
import functools

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from ..core import _native
from ..core import _DT, _ptr, _scratch, _stream

_REDUCTIONS = {'none': _native.REDUCE_NONE, 'mean': _native.REDUCE_MEAN, 'sum': _native.REDUCE_SUM}
_INDEX_BYTES = {torch.int64: 8, torch.int32: 4}
MAX_KEPT = 1024


def _reduction(name):
    if name not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {', '.join(_REDUCTIONS)}, got {name!r}")
    return _REDUCTIONS[name]


def _matrix(t, name):
    if t.dim() != 2:
        raise RuntimeError(f"{name} must be a matrix, got shape {tuple(t.shape)}")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if t.dtype not in _DT:
        raise RuntimeError(f"unsupported dtype {t.dtype} of {name}")


def _same_device(t, device, name):
    if t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, expected {device}")


def _rows_of(t):
    """``t`` with unit column stride and rows that do not overlap; what has neither is copied."""
    n, d = t.shape
    return t if (t.stride(1) == 1 or d == 1) and (t.stride(0) >= d or n == 1) and t.stride(0) > 0 else t.contiguous()


def _stride(t):
    """Row stride of a matrix of ``_rows_of`` (that of a single row means nothing)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _on(device, call):
    """``call()`` with ``device`` as the current device (a guard costs time: none where it is already)."""
    if torch.cuda.current_device() == device.index:
        return call()
    with torch.cuda.device(device):
        return call()


def _outputs(rows, per_row, reduction, device):
    """The loss and the state that goes to the backward call."""
    loss = torch.empty(rows if reduction == _native.REDUCE_NONE else (), dtype=torch.float32, device=device)
    state = torch.empty(rows * per_row + 4, dtype=torch.float32, device=device)      # the last four: the count of the rows
    return loss, state


@functools.lru_cache(maxsize=256)
def _ce_scratch_bytes(device_index, *args):
    return _native.lib().grws_linear_ce_scratch_bytes(*args)


def _ce_operands(x, w, class_major, V):
    """Leading arguments of the C calls, and the arguments that the size of their scratch depends on (where an operand
    starts matters to 16 bytes only)."""
    xp, wp, ldx, ldw = x.data_ptr(), w.data_ptr(), _stride(x), _stride(w)
    n, d = x.shape
    return (xp, ldx, wp, ldw, class_major), (x.device.index, 16 + xp % 16, ldx, 16 + wp % 16, ldw, class_major, n, d, V, _DT[x.dtype])


class _LinearCrossEntropyFunction(Function):
    @staticmethod
    def forward(ctx, x, weight, labels, ignore_index, reduction):
        x, labels = _rows_of(x), labels.contiguous()
        class_major = int(weight.stride(1) != 1 and weight.stride(0) == 1)
        w = _rows_of(weight.t() if class_major else weight)
        (n, d), V = x.shape, weight.shape[1]
        loss, state = _outputs(n, 2, reduction, x.device)

        def call():
            operands, key = _ce_operands(x, w, class_major, V)
            scratch = _scratch(_ce_scratch_bytes(*key, 0), x.device)
            sp = state.data_ptr()
            return _native.lib().grws_linear_ce_fwd(*operands, labels.data_ptr(), _INDEX_BYTES[labels.dtype], ignore_index, n, d, V, _DT[x.dtype],
                                                    reduction, loss.data_ptr(), sp, sp + 8 * n, scratch.data_ptr(), scratch.numel(),
                                                    _stream(x.device))
        _native.check(_on(x.device, call))
        ctx.save_for_backward(x, w, labels, state)
        ctx.args = (ignore_index, reduction, class_major, V)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss):
        x, w, labels, state = ctx.saved_tensors
        ignore_index, reduction, class_major, V = ctx.args
        n, d = x.shape
        grad_loss = grad_loss.contiguous()
        dx = torch.empty((n, d), dtype=x.dtype, device=x.device) if ctx.needs_input_grad[0] else None
        dw = torch.empty(w.shape, dtype=x.dtype, device=x.device) if ctx.needs_input_grad[1] else None

        def call():
            operands, key = _ce_operands(x, w, class_major, V)
            scratch = _scratch(_ce_scratch_bytes(*key, 1 if reduction == _native.REDUCE_NONE else 2), x.device)
            sp = state.data_ptr()
            return _native.lib().grws_linear_ce_bwd(*operands, labels.data_ptr(), _INDEX_BYTES[labels.dtype], ignore_index, n, d, V, _DT[x.dtype],
                                                    reduction, grad_loss.data_ptr(), sp, sp + 8 * n, _ptr(dx), _ptr(dw), scratch.data_ptr(),
                                                    scratch.numel(), _stream(x.device))
        _native.check(_on(x.device, call))
        return dx, dw.t() if class_major and dw is not None else dw, None, None, None


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, ignore_index: int = -100,
                         reduction: str = 'mean') -> torch.Tensor:
    """Softmax cross entropy of the scores ``x @ weight`` against ``labels``, without keeping the scores.

    x [rows, width] and weight [width, classes] (the layout of the layers' weights; the transpose of a
    [classes, width] matrix is as good) are fp32, fp16 or bf16 CUDA matrices of one type, labels [rows] int32 or
    int64.  Rows labelled ``ignore_index`` count nothing; any other label outside [0, classes) makes the loss
    and the gradients NaN.  'mean' divides by the number of counted rows (none: NaN, and no gradient),
    'none' returns a loss per row.  The backward pass computes the scores again, a piece of the classes
    at a time, and returns gradients of the operands' type; there is no second derivative.  Results do
    not change from call to call.

    Scores, softmax statistics, losses and all sums are fp32.  Of 16-bit operands the scores' gradient G is
    rounded to their type before the products with it, as a 16-bit layer's would be (fp16 without a
    reduction, where rows' gradients may be decades apart, keeps it to 24 bits and takes some four times as
    long).  Classes may be masked in the weight with the type's lowest value.  The gradient of the weight is
    ``x.T @ G``: an ignored row's part of it is 0 only if its ``x`` is finite.  The workspace of
    the backward pass holds G for as many classes as fit 512 MiB (256 at least, so more from a million
    rows on, in fp32 from 350,000) and fp32 sums of the gradients where they come in parts.  That of
    either pass holds copies of operands that the tensor cores do not read as they lie: unaligned
    rows, and fp32 as three bf16 planes (1.5 times its size)."""
    red = _reduction(reduction)
    _matrix(x, "x")
    _matrix(weight, "weight")
    if weight.dtype != x.dtype:
        raise RuntimeError(f"x is {x.dtype} and weight is {weight.dtype}: one dtype is expected")
    if weight.shape[0] != x.shape[1] or x.shape[1] == 0 or weight.shape[1] == 0:
        raise RuntimeError(f"x {tuple(x.shape)} and weight {tuple(weight.shape)} do not multiply to class scores")
    if labels.dtype not in _INDEX_BYTES:
        raise RuntimeError(f"labels must be int32 or int64, got {labels.dtype}")
    if tuple(labels.shape) != (x.shape[0],):
        raise RuntimeError(f"labels must have shape ({x.shape[0]},), got {tuple(labels.shape)}")
    _same_device(weight, x.device, "weight")
    _same_device(labels, x.device, "labels")
    return _LinearCrossEntropyFunction.apply(x, weight, labels, int(ignore_index), red)


@functools.lru_cache(maxsize=256)
def _distill_scratch_bytes(device_index, rows, classes):
    return _native.lib().grws_distill_scratch_bytes(rows, classes)


class _DistillationFunction(Function):
    @staticmethod
    def forward(ctx, logits, teacher, ids, temperature, reduction):
        logits, teacher, ids = _rows_of(logits), _rows_of(teacher), _rows_of(ids)
        (n, V), K = logits.shape, ids.shape[1]
        loss, state = _outputs(n, 4, reduction, logits.device)

        def call():
            scratch = _scratch(_distill_scratch_bytes(logits.device.index, n, V), logits.device)
            sp = state.data_ptr()
            return _native.lib().grws_distill_fwd(
                logits.data_ptr(), _stride(logits), _DT[logits.dtype], teacher.data_ptr(), _stride(teacher), _DT[teacher.dtype], ids.data_ptr(),
                _stride(ids), _INDEX_BYTES[ids.dtype], n, V, K, temperature, reduction, loss.data_ptr(), sp, sp + 16 * n, scratch.data_ptr(),
                scratch.numel(), _stream(logits.device))
        _native.check(_on(logits.device, call))
        ctx.save_for_backward(logits, teacher, ids, state)
        ctx.args = (temperature, reduction)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss):
        logits, teacher, ids, state = ctx.saved_tensors
        temperature, reduction = ctx.args
        (n, V), K = logits.shape, ids.shape[1]
        grad_loss = grad_loss.contiguous()
        # rows as far apart as the scores' (or, where these are a narrow cut, in whole 16-byte pieces), so that both
        # can be walked in the same 16-byte pieces
        ld = _stride(logits)
        ldo = ld if ld <= V + 16 else -(-V // 8) * 8
        dlogits = torch.empty((n, ldo), dtype=logits.dtype, device=logits.device)
        if ldo != V:
            dlogits = dlogits[:, :V]

        def call():
            sp = state.data_ptr()
            return _native.lib().grws_distill_bwd(
                logits.data_ptr(), ld, _DT[logits.dtype], teacher.data_ptr(), _stride(teacher), _DT[teacher.dtype], ids.data_ptr(), _stride(ids),
                _INDEX_BYTES[ids.dtype], n, V, K, temperature, reduction, grad_loss.data_ptr(), sp, sp + 16 * n, dlogits.data_ptr(), ldo,
                _stream(logits.device))
        _native.check(_on(logits.device, call))
        return dlogits, None, None, None, None


def distillation_loss(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_ids: torch.Tensor, temperature: float = 1.0,
                      reduction: str = 'mean') -> torch.Tensor:
    """``T^2 KL(p || softmax(logits / T))`` per row, in fp32, where p is the softmax over the teacher's kept scores at
    temperature T: a student learns the classes that its teacher finds best.

    logits [rows, classes] and teacher_logits [rows, kept] are fp32, fp16 or bf16 CUDA matrices, each of its own
    type, teacher_ids [rows, kept] the classes of the kept scores (int32 or int64, at most 1,024 a row).  An id
    below 0 is a missing entry, as padded column ids are, and a score of -inf has no weight; a row without
    entries of any weight counts nothing.  A class
    that occurs twice in a row counts with both scores; an id past the classes makes the row's loss
    and gradient NaN.  'mean' divides by the number of rows with entries (none: NaN, and no gradient), 'none'
    returns a loss per row.  Only ``logits`` has a gradient, and no second one.  A row's loss is the
    difference of two fp32 logarithms times T^2, off by some 2^-21 T^2: T in the hundreds leaves few digits of
    a loss of order 1."""
    red = _reduction(reduction)
    _matrix(logits, "logits")
    _matrix(teacher_logits, "teacher_logits")
    if teacher_ids.dtype not in _INDEX_BYTES:
        raise RuntimeError(f"teacher_ids must be int32 or int64, got {teacher_ids.dtype}")
    if teacher_ids.shape != teacher_logits.shape or teacher_ids.shape[0] != logits.shape[0]:
        raise RuntimeError(f"teacher_logits {tuple(teacher_logits.shape)} and teacher_ids {tuple(teacher_ids.shape)} must both be "
                           f"[{logits.shape[0]}, kept]")
    if logits.shape[1] == 0 or not 1 <= teacher_ids.shape[1] <= MAX_KEPT:
        raise RuntimeError(f"at least one class and between 1 and {MAX_KEPT} kept scores are expected, got {logits.shape[1]} and "
                           f"{teacher_ids.shape[1]}")
    _same_device(teacher_logits, logits.device, "teacher_logits")
    _same_device(teacher_ids, logits.device, "teacher_ids")
    if torch.is_grad_enabled() and teacher_logits.requires_grad:
        raise RuntimeError("teacher_logits gets no gradient: detach it")
    temperature = float(temperature)
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"temperature must lie between 1e-6 and 1e6, got {temperature}")
    return _DistillationFunction.apply(logits, teacher_logits, teacher_ids, temperature, red)
