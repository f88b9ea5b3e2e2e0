"""One training step of a small decoder whose parts run together: norm, packed projection, per-head norm
with rotation, flash attention, gated feed-forward, distillation from a teacher's top logits; and its
single-token forms against the full sequence.  The step is checked against the same model in 64 bits.

Tolerances: bf16 activations are rounded at every operator's border, about a dozen times on a path; each
rounding is 2^-8 of a value and enters the outputs and gradients at random signs, so the root mean square
error of a tensor stays below 12 * 2^-8 of its root mean square; the fp32 run (no native attention: head size
24) has only the sums' error, below 2^-12."""
import math

import pytest
import torch

from apex.contrib.xentropy import SoftmaxTopKDistillationLoss
from apex.fused_dense import fused_dense_gated_dense_function
from apex.normalization.fused_layer_norm import fused_rms_norm_affine
from apex.ops.attention import flash_attn_func
from apex.transformer.functional import fused_qk_norm_rope, rotary_tables

H, KVH, V, TOP = 4, 2, 307, 9


def _params(hid, d, f, dtype, dev):
    g = torch.Generator().manual_seed(5)
    rnd = lambda *s, std: (torch.randn(*s, generator=g) * std)
    p = dict(emb=rnd(V, hid, std=1.0), n1=1 + rnd(hid, std=0.1), qkv=rnd((H + 2 * KVH) * d, hid, std=hid ** -0.5),
             qn=1 + rnd(d, std=0.1), kn=1 + rnd(d, std=0.1), o=rnd(hid, H * d, std=(H * d) ** -0.5),
             n2=1 + rnd(hid, std=0.1), w1=rnd(2 * f, hid, std=hid ** -0.5), w2=rnd(hid, f, std=f ** -0.5))
    return {k: v.to(dtype).to(dev).requires_grad_(True) for k, v in p.items()}


def _project(p, x, b, s, d):
    qkv = (fused_rms_norm_affine(x, p["n1"], (x.size(-1),)) @ p["qkv"].t()).view(b, s, H + 2 * KVH, d)
    return qkv[:, :, :H], qkv[:, :, H:H + KVH], qkv[:, :, H + KVH:]


def _tail(p, x, ctx):
    x = x + ctx.flatten(2) @ p["o"].t()
    h = fused_rms_norm_affine(x, p["n2"], (x.size(-1),))
    return (x + fused_dense_gated_dense_function(h, p["w1"], None, p["w2"], None)) @ p["emb"].t()


def _forward(p, tok, pos, tables, d):
    b, s = tok.shape
    x = p["emb"][tok]
    q, k, v = _project(p, x, b, s, d)
    q, k = fused_qk_norm_rope(q, k, p["qn"], p["kn"], *tables, pos)
    return _tail(p, x, flash_attn_func(q, k, v, causal=True)), k, v


def _exact(p, tok, pos, tables, d, tz, ti, temp):
    p = {k: v.detach().double().cpu().requires_grad_(True) for k, v in p.items()}
    tok, pos, tz, ti = (t.cpu() for t in (tok, pos, tz, ti))
    cos, sin = (t.double().cpu()[pos].unsqueeze(-2) for t in tables)
    rms = lambda x, w, eps: x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w
    rot = lambda n: torch.cat((n[..., :d // 2] * cos - n[..., d // 2:] * sin,
                               n[..., d // 2:] * cos + n[..., :d // 2] * sin), -1)
    b, s = tok.shape
    x = p["emb"][tok]
    qkv = (rms(x, p["n1"], 1e-6) @ p["qkv"].t()).view(b, s, H + 2 * KVH, d)
    q, k, v = rot(rms(qkv[:, :, :H], p["qn"], 1e-6)), rot(rms(qkv[:, :, H:H + KVH], p["kn"], 1e-6)), qkv[:, :, H + KVH:]
    k, v = (t.repeat_interleave(H // KVH, 2).transpose(1, 2) for t in (k, v))
    sc = q.transpose(1, 2) @ k.transpose(-1, -2) / math.sqrt(d)
    sc = sc.masked_fill(torch.ones(s, s, dtype=torch.bool).triu(1), float("-inf"))
    x = x + (sc.softmax(-1) @ v).transpose(1, 2).flatten(2) @ p["o"].t()
    au = rms(x, p["n2"], 1e-6) @ p["w1"].t()
    a, u = au.chunk(2, -1)
    logits = (x + (torch.nn.functional.silu(a) * u) @ p["w2"].t()) @ p["emb"].t()
    live = ti >= 0
    t = torch.softmax((tz.double() / temp).masked_fill(~live, float("-inf")), -1).nan_to_num(0.0)
    lq = torch.log_softmax(logits.flatten(0, 1) / temp, -1).gather(1, ti.clamp(min=0))
    loss = (torch.where(t > 0, t * (t.clamp(min=1e-300).log() - lq), torch.zeros_like(t)).sum(-1) * temp ** 2).sum()
    loss.backward()
    return logits.detach(), loss.detach(), {k: v.grad for k, v in p.items()}


def _rms(t):
    return t.double().cpu().square().mean().sqrt().item()


def _run(dev, hid, d, f, dtype, tol):
    p = _params(hid, d, f, dtype, dev)
    g = torch.Generator().manual_seed(6)
    b, s, temp = 2, 37, 2.0
    tok = torch.randint(0, V, (b, s), generator=g).to(dev)
    pos = torch.arange(s).expand(b, s).to(dev)
    tables = rotary_tables(64, d, device=dev)
    tz, ti = (3 * torch.randn(b * s, V, generator=g)).topk(TOP, -1)
    ti[::7] = -1  # padding tokens
    ti[3, 4:] = -1
    tz, ti = tz.to(dev), ti.to(dev)
    logits, k, v = _forward(p, tok, pos, tables, d)
    losses = SoftmaxTopKDistillationLoss.apply(logits.flatten(0, 1), tz, ti, temp, True)
    assert (losses[::7] == 0).all()
    losses.sum().backward()
    want, loss, grads = _exact(p, tok, pos, tables, d, tz, ti, temp)
    assert _rms(logits.detach().double().cpu() - want) <= tol * _rms(want)
    assert abs(losses.sum().item() - loss.item()) <= tol * abs(loss.item())
    for name, w in p.items():
        assert _rms(w.grad.double().cpu() - grads[name]) <= tol * _rms(grads[name]), name

    # the last token alone, its key and value appended to the others': the same logits
    with torch.no_grad():
        x = p["emb"][tok[:, -1:]]
        q1, k1, v1 = _project(p, x, b, 1, d)
        q1, k1 = fused_qk_norm_rope(q1, k1, p["qn"], p["kn"], *tables, pos[:, -1:])
        kk, vv = torch.cat((k[:, :-1], k1), 1), torch.cat((v[:, :-1], v1), 1)
        last = _tail(p, x, flash_attn_func(q1, kk, vv))
        assert _rms(last[:, 0].double().cpu() - want[:, -1]) <= tol * _rms(want[:, -1])


def test_cpu_decoder_step():
    _run("cpu", 40, 24, 56, torch.float32, 2.0 ** -12)


@pytest.mark.gpu
def test_gpu_decoder_step_fp32():
    _run("cuda", 40, 24, 56, torch.float32, 2.0 ** -12)


@pytest.mark.gpu
@pytest.mark.parametrize("hid,d,f", [(64, 32, 136), (128, 64, 200)])
def test_gpu_decoder_step_bf16(hid, d, f):
    _run("cuda", hid, d, f, torch.bfloat16, 12 * 2.0 ** -8)
