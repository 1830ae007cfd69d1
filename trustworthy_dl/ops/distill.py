"""Distillation loss from a teacher's recorded top logits, mixed with cross-entropy.

``cross_entropy`` / ``lm_head_cross_entropy`` learn from labels alone.  ``distillation_loss`` learns
from the K largest logits that a teacher left for each token (indices and values), so no teacher pass
and no [tokens, vocab] teacher tensor is needed:

    kd_r = tau^2 KL(q_r || softmax(z_r / tau)),   q_r = softmax(t_r / tau) over the row's K entries
    loss = alpha mean(kd) + (1 - alpha) mean(cross-entropy)

GPU tensors run csrc/distill.hip: loss and gradient from one pass over the logits.  CPU tensors run
the same definition in PyTorch.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib

MAX_ENTRIES = 1024   # csrc/distill.hip MAX_K
MAX_DIM = (1 << 30) - 1   # csrc/distill.hip MAX_DIM - 1
MIN_TEMPERATURE, MAX_TEMPERATURE = 1e-6, 1000.0


class _Args(ctypes.Structure):
    """csrc/distill.hip DistillArgs"""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("logits", "grad", "index", "teacher", "labels", "gscale", "rows", "counts", "loss")]
                + [(n, ctypes.c_int64) for n in ("ld", "gld")]
                + [(n, ctypes.c_int) for n in ("M", "V", "W", "K", "G", "dtype", "index64", "teacher_dtype", "written")]
                + [("tau", ctypes.c_float), ("alpha", ctypes.c_float), ("beta", ctypes.c_float), ("capture", ctypes.c_uint64)])


def _rows(z: torch.Tensor) -> torch.Tensor:
    """``z`` [M, W] with unit column stride and rows that do not overlap: as it is, or a copy."""
    M, W = z.shape
    return z.contiguous() if z.stride(1) != 1 or (M > 1 and z.stride(0) < W) else z


def _grad_like(z: torch.Tensor) -> torch.Tensor:
    """Uninitialised [M, W] whose rows stand at the same offset from 16 bytes as the logits' rows."""
    M, W = z.shape
    per = 16 // z.element_size()
    ld = W + (z.stride(0) - W) % per if M > 1 else W
    skew = z.data_ptr() % 16 // z.element_size()
    if skew == 0:
        return torch.empty_strided((M, W), (ld, 1), dtype=z.dtype, device=z.device)
    return torch.empty(M * ld + skew, dtype=z.dtype, device=z.device)[skew:].as_strided((M, W), (ld, 1), skew)


def _alike(z: torch.Tensor, grad: torch.Tensor) -> bool:
    """``grad`` stands to the logits as _grad_like makes it."""
    return ((z.data_ptr() - grad.data_ptr()) % 16 == 0
            and (z.shape[0] == 1 or (z.stride(0) - grad.stride(0)) * z.element_size() % 16 == 0))


def _was(a: _Args, i: int):
    """(shape, type) of the i-th saved tensor"""
    types = {code: t for t, code in _lib.DTYPE_CODE.items()}
    return (((a.M, a.W), types[a.dtype]), ((a.M, a.K), torch.int64 if a.index64 else torch.int32), ((a.M, a.K), types[a.teacher_dtype]),
            ((a.M,), torch.int64), ((a.G, 2), torch.int32))[i]


class _Distill(torch.autograd.Function):
    """The forward leaves the gradient for an upstream gradient of 1 (loss.backward()); the backward
    launches a pass that reads the upstream gradient on the device and, where it is another, computes
    the gradient again from the logits (one rounding either way, no host synchronisation).  A backward
    captured into a graph without its forward always computes it."""

    @staticmethod
    def forward(ctx, z, index, teacher, labels, V, tau, alpha, grad):
        M = z.shape[0]
        dev = z.device
        rows = torch.empty(M, dtype=torch.float32, device=dev)
        loss = torch.empty((), dtype=torch.float32, device=dev)
        counts = torch.empty(max(1, min(256, -(-M // 256))), 2, dtype=torch.int32, device=dev)
        ctx.grad = _grad_like(z) if grad else None
        a = _Args(z.data_ptr(), 0, index.data_ptr(), teacher.data_ptr(), 0 if labels is None else labels.data_ptr(), 0, rows.data_ptr(),
                  counts.data_ptr(), loss.data_ptr(), z.stride(0), 0, M, V, z.shape[1], index.shape[1], counts.shape[0],
                  _lib.DTYPE_CODE[z.dtype], index.dtype is torch.int64, _lib.DTYPE_CODE[teacher.dtype], False, tau, alpha, 1.0 - alpha, 0)
        if grad:
            a.grad, a.gld = ctx.grad.data_ptr(), ctx.grad.stride(0)
        _lib.call_on(dev, "tdl_distill", ctypes.addressof(a))
        _lib.keep(ctx, z, index, teacher, labels, counts)
        ctx.args = a      # (and the graph capture that wrote the gradient)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        a = _Args.from_buffer_copy(ctx.args)
        z, index, teacher, labels, counts = _lib.came_back("distillation_loss", ctx, g.device, lambda i: _was(a, i),
                                                           lambda i, t: t.contiguous() if i else _rows(t))
        grad, ctx.grad = ctx.grad, None
        # a second backward through the same node gets its own buffer, and so do logits that saved-tensor
        # hooks brought back with other rows
        written = grad is not None and _alike(z, grad)
        if not written:
            grad = _grad_like(z)
        a.logits, a.ld, a.grad, a.gld = z.data_ptr(), z.stride(0), grad.data_ptr(), grad.stride(0)
        a.index, a.teacher, a.labels, a.counts = index.data_ptr(), teacher.data_ptr(), 0 if labels is None else labels.data_ptr(), counts.data_ptr()
        a.gscale, a.rows, a.loss, a.written = g.data_ptr(), 0, 0, written
        _lib.call_on(z.device, "tdl_distill", ctypes.addressof(a))
        return (grad,) + (None,) * 7


def _reference(z, index, teacher, labels, V, tau, alpha):
    wide = torch.float64 if z.dtype == torch.float64 else torch.float32
    zf, tf = z[:, :V].to(wide), teacher.to(wide)
    loss = zf.new_zeros(())
    if alpha > 0:
        has = ((index >= 0) & (index < V)).any(1)
        use = (index >= 0) & (index < V) & (tf != float("-inf"))
        t = torch.where(use, tf / tau, tf.new_full((), float("-inf")))
        top = torch.where(use.any(1, keepdim=True), t.amax(1, keepdim=True), t.new_zeros(()))
        e = torch.exp(t - top)
        total = e.sum(1, keepdim=True)
        total = torch.where(total == 0, torch.ones_like(total), total)
        q = e / total
        logq = torch.where(use, t - top, t.new_zeros(())) - torch.log(total)
        lp = torch.log_softmax(zf / tau, 1).gather(1, torch.where(use, index, 0).long())
        kd = torch.where(q != 0, q * (logq - lp), q.new_zeros(())).sum() * tau * tau
        loss = loss + alpha * kd / has.sum().clamp(min=1)
    if alpha < 1:
        ok = (labels >= 0) & (labels < V)
        lp = torch.log_softmax(zf, 1).gather(1, torch.where(ok, labels, 0)[:, None])[:, 0]
        loss = loss - (1 - alpha) * torch.where(ok, lp, lp.new_zeros(())).sum() / ok.sum().clamp(min=1)
    return loss


def distillation_loss(logits: torch.Tensor, teacher_index: torch.Tensor, teacher_logits: torch.Tensor,
                      labels: Optional[torch.Tensor] = None, num_classes: Optional[int] = None, *, temperature: float = 1.0,
                      alpha: float = 1.0) -> torch.Tensor:
    """``alpha`` x mean distillation + (1 - ``alpha``) x mean cross-entropy, an fp32 scalar.

    ``logits`` [..., W]: the student's, of which the first ``num_classes`` columns (default all) are
    classes and the rest padding, as in ``cross_entropy``.  ``teacher_index`` (int32 / int64) and
    ``teacher_logits`` [..., K], K <= 1024, in any order: an index outside [0, num_classes) marks an
    unused entry, a row without entries takes no part in the first mean (a row whose entries are all
    -inf counts, but has nothing to teach); an index that stands twice counts twice.  ``labels``
    (int32 / int64 [...], needed for alpha < 1): one outside [0, num_classes) takes no part in the second mean.
    ``temperature`` in [1e-6, 1000] (the first mean carries tau^2 times an error of 2^-20 or so).
    The gradient flows to ``logits`` (their type, zeros in the padding)."""
    if logits.dim() < 1 or not logits.dtype.is_floating_point:
        raise ValueError(f"distillation_loss: floating-point logits [..., classes], got {logits.dtype} {tuple(logits.shape)}")
    W = logits.shape[-1]
    V = W if num_classes is None else int(num_classes)
    if not 1 <= V <= W:
        raise ValueError(f"distillation_loss: num_classes must lie in [1, {W}], got {V}")
    if teacher_index.dim() == 0 or teacher_index.shape != teacher_logits.shape or teacher_index.shape[:-1] != logits.shape[:-1]:
        raise ValueError(f"distillation_loss: logits {tuple(logits.shape)}, teacher_index {tuple(teacher_index.shape)}, teacher_logits "
                         f"{tuple(teacher_logits.shape)} do not name the same rows")
    K = teacher_index.shape[-1]
    if not 1 <= K <= MAX_ENTRIES:
        raise ValueError(f"distillation_loss: 1 to {MAX_ENTRIES} teacher entries a row, got {K}")
    if teacher_index.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"distillation_loss: teacher_index must be int32 or int64, got {teacher_index.dtype}")
    if not teacher_logits.dtype.is_floating_point:
        raise ValueError(f"distillation_loss: teacher_logits must be floating-point, got {teacher_logits.dtype}")
    if teacher_logits.requires_grad:
        raise ValueError("distillation_loss: the teacher gets no gradient; pass teacher_logits.detach()")
    tau, alpha = float(temperature), float(alpha)
    if not MIN_TEMPERATURE <= tau <= MAX_TEMPERATURE:
        # (kd is tau^2 times a difference of logarithms in 32 bits: beyond this its rounding is all that is left; below
        # it 1 / tau would bring distances out of fp32's range)
        raise ValueError(f"distillation_loss: temperature must lie in [{MIN_TEMPERATURE:g}, {MAX_TEMPERATURE:g}], got {temperature}")
    if not 0 <= alpha <= 1:
        raise ValueError(f"distillation_loss: alpha must lie in [0, 1], got {alpha}")
    if alpha < 1:
        if labels is None:
            raise ValueError("distillation_loss: alpha < 1 needs labels")
        if labels.shape != logits.shape[:-1] or labels.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"distillation_loss: labels must be int32 or int64 {tuple(logits.shape[:-1])}, got {labels.dtype} {tuple(labels.shape)}")
    else:
        labels = None
    for name, t in (("teacher_index", teacher_index), ("teacher_logits", teacher_logits), ("labels", labels)):
        if t is not None and t.device != logits.device:
            raise ValueError(f"distillation_loss: {name} is on {t.device}, the logits on {logits.device}")
    z, index, teacher = logits, teacher_index, teacher_logits
    if z.dim() != 2:
        z, index, teacher = z.reshape(-1, W), index.reshape(-1, K), teacher.reshape(-1, K)
    labels = None if labels is None else labels.reshape(-1).long()
    if z.shape[0] == 0:
        return z.float().sum()   # no rows: zero, with a gradient of no rows
    if not z.is_cuda:
        return _reference(z, index, teacher, labels, V, tau, alpha)
    if z.dtype not in _lib.DTYPE_CODE:
        raise ValueError(f"native distillation_loss supports float32, bfloat16 and float16 logits (got {z.dtype})")
    if teacher.dtype not in _lib.DTYPE_CODE:
        raise ValueError(f"native distillation_loss supports float32, bfloat16 and float16 teacher logits (got {teacher.dtype})")
    if max(z.shape) > MAX_DIM:
        raise ValueError(f"native distillation_loss supports up to {MAX_DIM} rows and columns (got {tuple(z.shape)})")
    # (under no_grad an input that requires a gradient still counts as one that needs it)
    grad = z.requires_grad and torch.is_grad_enabled()
    return _Distill.apply(_rows(z), index.contiguous(), teacher.contiguous(), None if labels is None else labels.contiguous(), V, tau, alpha,
                          grad)
