"""Gated feed-forward block: ``y = (act(x Wg^T + bg) * (x Wu^T + bu)) W2^T + b2``.

``weight1`` ``[2 * intermediate, in]`` holds the gate rows ``Wg``, then the up rows ``Wu`` (``bias1``
likewise), ``weight2`` is ``[out, intermediate]``; the activation is ``silu`` or ``gelu`` (tanh form, as
:class:`FusedDenseGeluDense`).  fp16 / bf16 GPU tensors with widths that are multiples of 8 run the gfx950
kernels of ``csrc/gemm/gated_ffn.hip``: both projections, the activation and the product are one MFMA
kernel, the backward's ``[da | du]`` another, and no operand is transposed or concatenated in memory
(differentiable once: ``create_graph`` is refused).
Other types and widths (CPU, fp32, odd sizes) run the same math in torch, as the other fused dense layers."""
import torch
from torch import nn

from .. import _native
from .._autocast_utils import _active_device, _autocast_disabled, _cast_if_autocast_enabled
from ..amp import half_function

_ACTIVATIONS = ("silu", "gelu")


def _ext():
    return _native.require("gated_ffn").gated_ffn


def _check(x, w1, b1, w2, b2, activation):
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {_ACTIVATIONS}, got {activation!r}")
    if w1.dim() != 2 or w2.dim() != 2 or w1.size(0) != 2 * w2.size(1) or w2.size(1) == 0:
        raise ValueError(f"weight1 [2 * intermediate, in] and weight2 [out, intermediate] expected, got "
                         f"{tuple(w1.shape)} and {tuple(w2.shape)}")
    if x.dim() < 1 or x.size(-1) != w1.size(1):
        raise ValueError(f"input [..., {w1.size(1)}] expected, got {tuple(x.shape)}")
    for b, n, what in ((b1, w1.size(0), "bias1"), (b2, w2.size(0), "bias2")):
        if b is not None and tuple(b.shape) != (n,):
            raise ValueError(f"{what} must be [{n}], got {tuple(b.shape)}")
    ts = [t for t in (w1, b1, w2, b2) if t is not None]
    if any(t.device != x.device for t in ts):
        raise ValueError("input, weights and biases must be on one device")
    if any(t.dtype != x.dtype for t in ts) or not x.is_floating_point():
        raise TypeError("input, weights and biases must have one floating-point dtype")


def _native_ok(x, w1, w2):
    return (_native.use_native(x) and x.dtype in (torch.float16, torch.bfloat16) and x.size(-1) % 8 == 0
            and w2.size(0) % 8 == 0 and w2.size(1) % 8 == 0 and x.size(-1) > 0 and w2.size(0) > 0)


def _torch_gated_dense(x, w1, b1, w2, b2, activation):
    au = torch.nn.functional.linear(x, w1, b1)
    a, u = au.chunk(2, dim=-1)
    act = torch.nn.functional.silu(a) if activation == "silu" else torch.nn.functional.gelu(a, approximate="tanh")
    return torch.nn.functional.linear(act * u, w2, b2)


def _gated_dense(input, weight1, bias1, weight2, bias2, activation="silu"):
    """:func:`fused_dense_gated_dense_function`: ``(input, weight1, bias1, weight2, bias2, activation)``, the
    biases ``None`` where there are none.  Under autocast the tensors are cast to its dtype."""
    if _active_device() is not None:
        args = _cast_if_autocast_enabled(input, weight1, bias1, weight2, bias2)
        with _autocast_disabled():
            return _gated_dense(*args, activation)
    _check(input, weight1, bias1, weight2, bias2, activation)
    if not _native_ok(input, weight1, weight2):
        return _torch_gated_dense(input, weight1, bias1, weight2, bias2, activation)
    ext = _ext()
    y = ext.gated_ffn(input.reshape(-1, input.size(-1)), weight1, bias1, weight2, bias2,
                      ext.ACT_SILU if activation == "silu" else ext.ACT_GELU)
    return y if input.dim() == 2 else y.view(input.shape[:-1] + (weight2.size(0),))


fused_dense_gated_dense_function = half_function(_gated_dense)


class FusedDenseGatedDense(nn.Module):
    """The gated feed-forward block as a module: ``weight1`` is ``[2 * intermediate_features, in_features]``
    (gate rows, then up rows), ``weight2`` ``[out_features, intermediate_features]``."""

    def __init__(self, in_features, intermediate_features, out_features, bias=False, activation="silu"):
        super().__init__()
        if activation not in _ACTIVATIONS:
            raise ValueError(f"activation must be one of {_ACTIVATIONS}, got {activation!r}")
        self.in_features = in_features
        self.intermediate_features = intermediate_features
        self.out_features = out_features
        self.activation = activation
        self.weight1 = nn.Parameter(torch.empty(2 * intermediate_features, in_features))
        self.weight2 = nn.Parameter(torch.empty(out_features, intermediate_features))
        if bias:
            self.bias1 = nn.Parameter(torch.empty(2 * intermediate_features))
            self.bias2 = nn.Parameter(torch.empty(out_features))
        else:
            self.register_parameter("bias1", None)
            self.register_parameter("bias2", None)
        self.reset_parameters()

    def reset_parameters(self):
        for w, b, fan_in in ((self.weight1, self.bias1, self.in_features),
                             (self.weight2, self.bias2, self.intermediate_features)):
            nn.init.kaiming_uniform_(w, a=5 ** 0.5)
            if b is not None:
                nn.init.uniform_(b, -1 / fan_in ** 0.5, 1 / fan_in ** 0.5)

    def forward(self, input):
        return fused_dense_gated_dense_function(input, self.weight1, self.bias1, self.weight2, self.bias2,
                                                self.activation)

    def extra_repr(self):
        return (f"in_features={self.in_features}, intermediate_features={self.intermediate_features}, "
                f"out_features={self.out_features}, bias={self.bias1 is not None}, activation={self.activation!r}")
