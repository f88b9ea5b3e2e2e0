"""RMS norm of every query / key head and the rotary position rotation, in one pass.

    n = x * rsqrt(mean(x^2) + eps) * weight          over each head
    (y1, y2) = (n1 cos - n2 sin, n2 cos + n1 sin)    for the rotated pairs of the head

GPU (fp16 / bf16 / fp32): one gfx950 kernel each way for queries and keys together
(``csrc/transformer/qk_norm_rope.hip``); everything between the load and the store of an element is
fp32, and the norm weights' gradients are fixed-order sums.  CPU: the same math in torch.
The outputs feed :func:`apex.ops.attention.flash_attn_func`; a single token of a running sequence is
the same call with that token's position."""
import torch

from ... import _native

_MAX_HEAD = 512


def rotary_tables(max_positions, rotary_dim, base=10000.0, device=None):
    """fp32 ``(cos, sin)`` tables ``[max_positions, rotary_dim / 2]`` of the angles
    ``position * base ** (-2 i / rotary_dim)``, computed in 64 bits (a far position's angle has more
    digits than fp32 holds)."""
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even, got {rotary_dim}")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device)
    inv = base ** (-i / max(rotary_dim, 1))
    ang = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def _torch_qk_norm_rope(x, weight, cos, sin, positions, eps, interleaved):
    acc = torch.promote_types(x.dtype, torch.float32)
    xf = x.to(acc)
    n = xf * torch.rsqrt((xf * xf).mean(-1, keepdim=True) + eps)
    if weight is not None:
        n = n * weight.to(acc).reshape(-1)
    rot = 2 * cos.size(1)
    bad = (positions < 0) | (positions >= cos.size(0))
    pos = torch.where(bad, torch.zeros_like(positions), positions)
    c, s = cos[pos].unsqueeze(-2).to(acc), sin[pos].unsqueeze(-2).to(acc)
    if interleaved:
        a, b = n[..., 0:rot:2], n[..., 1:rot:2]
        y = torch.stack((a * c - b * s, b * c + a * s), dim=-1).flatten(-2)
    else:
        a, b = n[..., :rot // 2], n[..., rot // 2:rot]
        y = torch.cat((a * c - b * s, b * c + a * s), dim=-1)
    y = torch.cat((y, n[..., rot:]), dim=-1)
    # a factor of NaN rather than a fill: the gradient of such a row is NaN too
    return (y * torch.where(bad, float("nan"), 1.0).to(acc)[..., None, None]).to(x.dtype)


def _rows(t):
    """Last dimension contiguous (the kernels take any other strides)."""
    return t if t.stride(-1) == 1 or t.size(-1) == 1 else t.contiguous()


def fused_qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps=1e-6, interleaved=False):
    """Normed and rotated ``(q', k')`` of queries ``[..., heads, d]`` and keys ``[..., kv_heads, d]``
    (one or two leading token axes, the same for both; any strides with d contiguous, e.g. views of a
    packed projection).  The outputs are contiguous.

    ``q_weight`` / ``k_weight``: ``[d]`` norm weights, both or neither (None), fp32 or the inputs'
    dtype.  ``cos`` / ``sin``: fp32 tables ``[positions, rotary_dim / 2]`` (:func:`rotary_tables`);
    ``rotary_dim`` may be smaller than the head, the rest of the head is then normed only.
    ``positions``: integers, broadcastable to the token axes; a position outside the table makes that
    token's output (and gradients) NaN.  ``interleaved`` rotates the pairs ``(2i, 2i + 1)`` instead of
    ``(i, i + rotary_dim / 2)``.  The head size is even, up to 512 on the GPU, where the operator is
    differentiable once (``create_graph`` is refused)."""
    if q.dim() not in (3, 4) or q.dim() != k.dim() or q.shape[:-2] != k.shape[:-2] or q.size(-1) != k.size(-1):
        raise ValueError(f"q and k must be [..., heads, d] with the same one or two token axes and d, got "
                         f"{tuple(q.shape)} and {tuple(k.shape)}")
    if q.dtype != k.dtype or not q.is_floating_point():
        raise TypeError(f"q and k must have one floating-point dtype, got {q.dtype} and {k.dtype}")
    d = q.size(-1)
    if d < 2 or d % 2:
        raise ValueError(f"the head size must be even, got {d}")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("give both norm weights or neither")
    for w in (q_weight, k_weight):
        if w is not None and (w.numel() != d or w.dtype not in (torch.float32, q.dtype) or w.dtype != q_weight.dtype):
            raise ValueError(f"norm weights must be [{d}], both fp32 or both {q.dtype}")
    if cos.dim() != 2 or cos.shape != sin.shape or 2 * cos.size(1) > d:
        raise ValueError(f"cos and sin must be [positions, rotary_dim / 2] tables with rotary_dim <= {d}, got "
                         f"{tuple(cos.shape)} and {tuple(sin.shape)}")
    if positions.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"positions must be int64 or int32, got {positions.dtype}")
    if cos.requires_grad or sin.requires_grad:
        raise ValueError("the rotary tables take no gradient")
    tensors = [t for t in (k, q_weight, k_weight, cos, sin, positions) if t is not None]
    if any(t.device != q.device for t in tensors):
        raise ValueError("q, k, the weights, the tables and the positions must be on one device")
    positions = positions.expand(q.shape[:-2])
    if cos.size(0) == 0 and positions.numel():
        raise ValueError("the rotary tables are empty")
    if not _native.use_native(q):
        return (_torch_qk_norm_rope(q, q_weight, cos, sin, positions, eps, interleaved),
                _torch_qk_norm_rope(k, k_weight, cos, sin, positions, eps, interleaved))
    if q.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise TypeError(f"fp16, bf16 or fp32 queries and keys expected on the GPU, got {q.dtype}")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise TypeError("the rotary tables must be fp32")
    if d > _MAX_HEAD:
        raise ValueError(f"the head size must be at most {_MAX_HEAD}, got {d}")
    flat = q.dim() == 3
    if flat:
        q, k, positions = q.unsqueeze(0), k.unsqueeze(0), positions.unsqueeze(0)
    ext = _native.require("fused_transformer").fused_transformer
    qo, ko = ext.qk_norm_rope(_rows(q), _rows(k), q_weight, k_weight, cos, sin, positions, float(eps),
                              bool(interleaved))
    return (qo[0], ko[0]) if flat else (qo, ko)
