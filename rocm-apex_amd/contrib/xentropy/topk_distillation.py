"""Distillation loss against a teacher's top logits.

``SoftmaxTopKDistillationLoss.apply(logits, teacher_logits, teacher_indices, temperature=1.0,
half_to_float=False)`` returns per-row losses

    T^2 * sum_k t_k (log t_k - log softmax(logits / T)[index_k]),   t = softmax(teacher_logits / T)

of student ``logits`` ``[rows, classes]`` and the ``top`` largest logits the teacher kept of each row
(``[rows, top]`` values and int64 / int32 class indices, the teacher's probabilities renormalised over
them).  An entry with a negative index is no entry (a row may keep fewer); a row without entries (or
whose teacher logits are all -inf) has zero loss and zero gradient, whatever its logits hold.  Entries naming
one class twice both count.  An index past the classes makes the row's loss and gradient NaN.  The
teacher is a constant: it takes no gradient.  Temperatures are between 1e-15 and 1e15.  The loss is differentiable once (``create_graph`` is refused).

GPU: the gfx950 kernels of ``csrc/xentropy/topk_distill.hip`` (the logits are read once forward and
once backward, in place for any row pitch); CPU: the same math in torch.  Like
:class:`~apex.contrib.xentropy.SoftmaxCrossEntropyLoss`, losses come in the logits' dtype unless
``half_to_float``."""
import torch

from ... import _native

_MAX_TOP = 1024


def _ext():
    return _native.require("xentropy_cuda").xentropy_cuda


def _check(logits, teacher_logits, teacher_indices, temperature):
    if logits.dim() != 2 or logits.size(1) == 0 or not logits.is_floating_point():
        raise ValueError(f"floating-point logits [rows, classes] expected, got {tuple(logits.shape)} {logits.dtype}")
    if teacher_logits.dim() != 2 or teacher_logits.shape != teacher_indices.shape \
            or teacher_logits.size(0) != logits.size(0):
        raise ValueError(f"teacher logits and indices must both be [{logits.size(0)}, top], got "
                         f"{tuple(teacher_logits.shape)} and {tuple(teacher_indices.shape)}")
    if not teacher_logits.is_floating_point() or teacher_indices.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"floating-point teacher logits and int64 / int32 indices expected, got "
                        f"{teacher_logits.dtype} and {teacher_indices.dtype}")
    if teacher_logits.device != logits.device or teacher_indices.device != logits.device:
        raise ValueError("the teacher's logits and indices must be on the logits' device")
    # 1 / T and T^2 are fp32 factors of the kernels' exponents and losses
    if not 1e-15 <= temperature <= 1e15:
        raise ValueError(f"the temperature must be between 1e-15 and 1e15, got {temperature}")
    if _native.use_native(logits):
        if logits.dtype not in (torch.float16, torch.bfloat16, torch.float32):
            raise TypeError(f"fp16, bf16 or fp32 logits expected on the GPU, got {logits.dtype}")
        if teacher_logits.size(1) > _MAX_TOP:
            raise ValueError(f"at most {_MAX_TOP} teacher entries a row, got {teacher_logits.size(1)}")


def _torch_teacher(teacher_logits, teacher_indices, temperature, classes, acc):
    """(t, T log t, index clamped to the classes, rows with entries, rows with a bad index)."""
    live = (teacher_indices >= 0) & (teacher_indices < classes)
    bad = (teacher_indices >= classes).any(-1)
    z = teacher_logits.to(acc).masked_fill(~live, float("-inf"))
    if z.size(1) == 0:
        return z, z, teacher_indices.long(), bad, bad
    zm = z.amax(-1, keepdim=True)
    z = z - torch.where(torch.isinf(zm) & (zm < 0), torch.zeros_like(zm), zm)
    total = torch.exp(z / temperature).sum(-1, keepdim=True)
    some = total.squeeze(-1) != 0
    total = torch.where(total != 0, total, torch.ones_like(total))
    t = torch.where(some[:, None], torch.exp(z / temperature) / total, torch.zeros_like(z))
    tlogt = z - temperature * torch.log(total)
    return t, tlogt, torch.where(live, teacher_indices, torch.zeros_like(teacher_indices)).long(), some, bad


def _torch_student(logits, acc):
    # the maximum goes first: logits of the type's lowest value over a temperature below 1 are no numbers of acc
    x = logits.to(acc)
    return x - x.amax(-1, keepdim=True)


def _torch_forward(logits, teacher_logits, teacher_indices, temperature):
    acc = torch.promote_types(logits.dtype, torch.float32)
    t, tlogt, idx, some, bad = _torch_teacher(teacher_logits, teacher_indices, temperature, logits.size(1), acc)
    # T log q: log q of such a logit overflows where its term of the loss does not
    x = _torch_student(logits, acc)
    tlogq = x.gather(1, idx) - temperature * torch.logsumexp(x / temperature, -1, keepdim=True)
    terms = torch.where(t != 0, t * (tlogt - tlogq), torch.zeros_like(t)).sum(-1) * temperature
    terms = torch.where(some, terms, torch.zeros_like(terms))
    return terms.masked_fill(bad, float("nan"))


def _torch_backward(grad_loss, logits, teacher_logits, teacher_indices, temperature):
    acc = torch.promote_types(logits.dtype, torch.float32)
    t, _, idx, some, bad = _torch_teacher(teacher_logits, teacher_indices, temperature, logits.size(1), acc)
    q = torch.softmax(_torch_student(logits, acc) / temperature, -1)
    g = (grad_loss.to(acc) * temperature).masked_fill(bad, float("nan"))[:, None]
    dx = g * q.scatter_add(1, idx, -t)
    return torch.where((some | bad)[:, None], dx, torch.zeros_like(dx)).to(logits.dtype)


class _TorchTopKDistillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher_logits, teacher_indices, temperature, half_to_float):
        ctx.save_for_backward(logits, teacher_logits, teacher_indices)
        ctx.temperature = temperature
        losses = _torch_forward(logits, teacher_logits, teacher_indices, temperature)
        return losses if half_to_float else losses.to(logits.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        return _torch_backward(grad_loss, *ctx.saved_tensors, ctx.temperature), None, None, None, None


class SoftmaxTopKDistillationLoss:
    """See the module's documentation; used through :meth:`apply` like the other losses here."""

    @staticmethod
    def apply(logits, teacher_logits, teacher_indices, temperature=1.0, half_to_float=False):
        temperature = float(temperature)
        _check(logits, teacher_logits, teacher_indices, temperature)
        if teacher_logits.requires_grad and torch.is_grad_enabled():
            raise ValueError("the teacher takes no gradient: detach its logits")
        if _native.use_native(logits):
            return _ext().topk_distill(logits, teacher_logits, teacher_indices, temperature, bool(half_to_float))
        return _TorchTopKDistillation.apply(logits, teacher_logits, teacher_indices, temperature, bool(half_to_float))
