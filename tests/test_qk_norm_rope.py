"""Per-head RMS norm + rotary rotation of queries and keys, against the formulas in 64 bits.

Tolerances: one rounding of the result to its type is eps/2 of the value.  The fp32 arithmetic before it
(mean of d squares, rsqrt, two products, one rotation: each term a few 2^-24 of the row's largest
magnitudes) is bounded by 16 * 2^-23 of the row's largest value for d <= 512; weights' gradients
are sums of n terms, bounded by n_terms-independent pairwise order here only through their 64-bit
sum of magnitudes: (32 + sqrt(n)) * 2^-24 of it."""
import pytest
import torch

from apex.transformer.functional import fused_qk_norm_rope, rotary_tables


def _exact(x, w, cos, sin, pos, eps, inter, dy=None):
    """(y, dx, dw) in 64 bits, written out pair by pair."""
    x, cos, sin = x.detach().double(), cos.double(), sin.double()
    half, d = cos.size(1), x.size(-1)
    w = torch.ones(d, dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    i = torch.arange(half, device=x.device)
    first, second = (2 * i, 2 * i + 1) if inter else (i, i + half)
    pos = pos.expand(x.shape[:-2])
    c, s = cos[pos].unsqueeze(-2), sin[pos].unsqueeze(-2)
    r = (x.square().mean(-1, keepdim=True) + eps).pow(-0.5)
    n = x * r * w
    y = n.clone()
    y[..., first] = n[..., first] * c - n[..., second] * s
    y[..., second] = n[..., second] * c + n[..., first] * s
    if dy is None:
        return y, None, None, None
    dy = dy.double()
    dn = dy.clone()
    dn[..., first] = dy[..., first] * c + dy[..., second] * s
    dn[..., second] = dy[..., second] * c - dy[..., first] * s
    xh = x * r
    gw = dn * w
    dx = r * (gw - xh * (gw * xh).mean(-1, keepdim=True))
    terms = (dn * xh).flatten(0, -2)
    return y, dx, terms.sum(0), terms.abs().sum(0)


def _close(got, want, what):
    eps = torch.finfo(got.dtype).eps
    scale = want.abs().amax(-1, keepdim=True)
    # fp16 results near zero are rounded in steps of 2^-24
    tiny = 2.0 ** -24 if got.dtype == torch.float16 else 0.0
    bound = eps / 2 * 1.01 * want.abs() + 16 * 2.0 ** -23 * scale + tiny
    bad = (got.double() - want).abs() > bound
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst " \
                          f"{float(((got.double() - want).abs() / bound).max()):.2f} bounds"


def _close_dw(got, want, mag, rows, what):
    eps = torch.finfo(got.dtype).eps
    bound = eps / 2 * 1.01 * want.abs() + (32 + rows ** 0.5) * 2.0 ** -24 * mag
    assert ((got.double() - want).abs() <= bound).all(), what


def _case(dev, lead, hq, hk, d, rot, inter, dtype, wdtype, packed, seed=0, table=97):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)
    if packed:
        mixed = (2 * rnd(*lead, hq + 2 * hk, d)).to(dtype).to(dev)
        q, k = mixed[..., :hq, :], mixed[..., hq:hq + hk, :]
    else:
        q, k = (2 * rnd(*lead, hq, d)).to(dtype).to(dev), (2 * rnd(*lead, hk, d)).to(dtype).to(dev)
    qw = kw = None
    if wdtype is not None:
        qw, kw = ((1 + 0.3 * rnd(d)).to(wdtype).to(dev).requires_grad_(True) for _ in range(2))
    cos, sin = rotary_tables(table, rot, device=dev)
    pos = torch.randint(0, table, lead, generator=g).to(dev)
    gq, gk = rnd(*lead, hq, d).to(dtype).to(dev), rnd(*lead, hk, d).to(dtype).to(dev)
    return q.detach().requires_grad_(True), k.detach().requires_grad_(True), qw, kw, cos, sin, pos, gq, gk


def _check_case(c, eps, inter):
    q, k, qw, kw, cos, sin, pos, gq, gk = c
    qo, ko = fused_qk_norm_rope(q, k, qw, kw, cos, sin, pos, eps, inter)
    assert qo.is_contiguous() and ko.is_contiguous() and qo.dtype == q.dtype and qo.shape == q.shape
    leaves = [q, k] + ([qw, kw] if qw is not None else [])
    grads = torch.autograd.grad((qo, ko), leaves, (gq, gk))
    rows = q.numel() // q.size(-1) * max(1, k.size(-2) // max(q.size(-2), 1))
    for i, (x, o, w, g) in enumerate(((q, qo, qw, gq), (k, ko, kw, gk))):
        y, dx, dw, mag = _exact(x, w, cos, sin, pos, eps, inter, g)
        _close(o.detach(), y, "qk"[i])
        _close(grads[i], dx, "d" + "qk"[i])
        if w is not None:
            _close_dw(grads[2 + i], dw, mag, rows, "dw" + "qk"[i])


SHAPES = [  # lead, hq, hk, d, rot
    ((5,), 4, 4, 64, 64), ((3, 2), 4, 2, 128, 128), ((1, 1), 1, 1, 2, 2), ((7,), 3, 1, 80, 32),
    ((1, 9), 5, 5, 72, 72), ((2, 3), 6, 2, 96, 0), ((4,), 2, 2, 256, 64), ((2, 2), 2, 1, 34, 18), ((3,), 7, 7, 512, 512),
    ((2,), 1, 3, 130, 66), ((3,), 2, 1, 400, 398), ((5,), 3, 2, 200, 8), ((31,), 7, 2, 144, 52), ((2, 9), 3, 1, 176, 160),
]


@pytest.mark.parametrize("lead,hq,hk,d,rot", SHAPES)
@pytest.mark.parametrize("inter", [False, True])
def test_cpu_qk_norm_rope(lead, hq, hk, d, rot, inter):
    for dtype, wdtype in ((torch.float32, torch.float32), (torch.bfloat16, None), (torch.bfloat16, torch.bfloat16)):
        _check_case(_case("cpu", lead, hq, hk, d, rot, inter, dtype, wdtype, len(lead) == 2), 1e-6, inter)


def test_cpu_gradient_against_differences():
    q, k, qw, kw, cos, sin, pos, _, _ = _case("cpu", (2,), 2, 1, 6, 4, False, torch.float64, torch.float64, False)
    f = lambda q, k, qw, kw: fused_qk_norm_rope(q, k, qw, kw, cos, sin, pos, 1e-3)
    assert torch.autograd.gradcheck(f, (q, k, qw, kw))


def test_rotary_tables_keep_far_positions():
    cos, sin = rotary_tables(131072, 128)
    ang = torch.tensor(131071.0, dtype=torch.float64) * 10000.0 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128)
    assert cos.dtype == torch.float32 and cos.shape == (131072, 64)
    assert (cos[-1].double() - ang.cos()).abs().max() <= 2.0 ** -24
    assert (sin[-1].double() - ang.sin()).abs().max() <= 2.0 ** -24


def _refusals(dev):
    mk = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device=dev)
    cos, sin = rotary_tables(8, 16, device=dev)
    pos = torch.zeros(3, dtype=torch.int64, device=dev)
    ok = dict(q=mk(3, 2, 16), k=mk(3, 1, 16), q_weight=None, k_weight=None, cos=cos, sin=sin, positions=pos)
    fused_qk_norm_rope(**ok)
    bad = [
        (ValueError, dict(q=mk(3, 2, 15), k=mk(3, 1, 15))), (ValueError, dict(k=mk(4, 1, 16))),
        (ValueError, dict(q=mk(16), k=mk(16))), (ValueError, dict(k=mk(3, 1, 8))),
        (TypeError, dict(k=mk(3, 1, 16, dt=torch.bfloat16))), (ValueError, dict(q_weight=mk(16))),
        (ValueError, dict(q_weight=mk(8), k_weight=mk(8))),
        (ValueError, dict(q_weight=mk(16), k_weight=mk(16, dt=torch.bfloat16))),
        (ValueError, dict(cos=mk(8, 16), sin=mk(8, 16))), (ValueError, dict(sin=mk(7, 8))),
        (ValueError, dict(cos=mk(0, 8), sin=mk(0, 8))), (TypeError, dict(positions=pos.float())),
        (RuntimeError, dict(positions=torch.zeros(2, dtype=torch.int64, device=dev))),
        (ValueError, dict(cos=cos.clone().requires_grad_(True))),
    ]
    for err, change in bad:
        with pytest.raises(err):
            fused_qk_norm_rope(**{**ok, **change})


def test_cpu_refusals():
    _refusals("cpu")
    with pytest.raises(ValueError):
        rotary_tables(8, 15)


def _bad_positions(dev):
    q, k, qw, kw, cos, sin, pos, gq, gk = _case(dev, (4,), 2, 2, 32, 16, False, torch.float32, torch.float32, False)
    pos = torch.tensor([0, -1, 97, 96], device=dev)
    qo, ko = fused_qk_norm_rope(q, k, qw, kw, cos, sin, pos)
    for o in (qo, ko):
        assert o[1:3].isnan().all() and o[0].isfinite().all() and o[3].isfinite().all()
    dq, = torch.autograd.grad(qo, q, gq)
    assert dq[1:3].isnan().all() and dq[0].isfinite().all() and dq[3].isfinite().all()


def test_cpu_bad_positions_are_nan_rows():
    _bad_positions("cpu")


# ------------------------------------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("lead,hq,hk,d,rot", SHAPES + [((257, 3), 8, 2, 128, 128), ((2100,), 16, 16, 64, 64),
                                                       ((1, 700), 12, 4, 80, 36), ((40, 33), 5, 3, 96, 96)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                          (torch.bfloat16, torch.bfloat16), (torch.float16, None),
                                          (torch.float16, torch.float16)])
def test_gpu_qk_norm_rope(lead, hq, hk, d, rot, inter, dtype, wdtype):
    _check_case(_case("cuda", lead, hq, hk, d, rot, inter, dtype, wdtype, len(lead) == 2), 1e-6, inter)


@pytest.mark.gpu
def test_gpu_refusals():
    _refusals("cuda")
    z = lambda *s: torch.zeros(*s, device="cuda")
    cos, sin = rotary_tables(8, 16, device="cuda")
    pos = torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError):
        fused_qk_norm_rope(z(3, 1, 514), z(3, 1, 514), None, None, cos, sin, pos)
    with pytest.raises(ValueError):
        fused_qk_norm_rope(z(3, 1, 16), z(3, 1, 16), None, None, cos, sin, pos.cpu())
    with pytest.raises(TypeError):
        fused_qk_norm_rope(z(3, 1, 16).double(), z(3, 1, 16).double(), None, None, cos, sin, pos)
    with pytest.raises(TypeError):
        fused_qk_norm_rope(z(3, 1, 16), z(3, 1, 16), None, None, cos.half(), sin.half(), pos)


@pytest.mark.gpu
def test_gpu_bad_positions_are_nan_rows():
    _bad_positions("cuda")


@pytest.mark.gpu
def test_gpu_empty_and_single():
    cos, sin = rotary_tables(8, 32, device="cuda")
    w = torch.ones(32, device="cuda", requires_grad=True)
    q = torch.zeros(0, 4, 32, device="cuda", requires_grad=True)
    pos = torch.zeros(0, dtype=torch.int32, device="cuda")
    qo, ko = fused_qk_norm_rope(q, q, w, w, cos, sin, pos)
    assert qo.shape == (0, 4, 32)
    (qo.sum() + ko.sum()).backward()
    assert (w.grad == 0).all() and q.grad.shape == q.shape
    # a row of zeros stays zero; its gradient is finite
    z = torch.zeros(1, 1, 32, device="cuda", requires_grad=True)
    zo, _ = fused_qk_norm_rope(z, z, None, None, cos, sin, torch.tensor([3], device="cuda"))
    assert (zo == 0).all()
    zo.sum().backward()
    assert z.grad.isfinite().all()


@pytest.mark.gpu
def test_gpu_strides_broadcast_gradients_and_repeatability():
    dev = "cuda"
    base = torch.randn(6, 5, 4, 3 * 64, device=dev).to(torch.bfloat16)
    q, k = base[..., 3:67].requires_grad_(True), base.transpose(0, 1)[..., 64:128].transpose(0, 1)
    cos, sin = rotary_tables(50, 64, device=dev)
    pos = torch.arange(6, device=dev, dtype=torch.int32)[:, None]  # broadcast over the batch
    w = torch.ones(64, device=dev, requires_grad=True)
    qo, ko = fused_qk_norm_rope(q, k, w, w, cos, sin, pos)
    y, dx, _, _ = _exact(q, w, cos, sin, pos.long(), 1e-6, False, torch.ones_like(qo))
    _close(qo.detach(), y, "q")
    _close(ko.detach(), _exact(k, w, cos, sin, pos.long(), 1e-6, False)[0], "k")
    g1 = torch.autograd.grad(qo.sum(), [q, w], retain_graph=True)  # an expanded gradient, none for k
    _close(g1[0], dx, "dq")
    g2 = torch.autograd.grad(qo.sum(), [q, w], retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(g1, g2))


@pytest.mark.gpu
def test_gpu_other_stream_and_captured_graph():
    c = _case("cuda", (130, 2), 8, 2, 128, 64, False, torch.bfloat16, torch.float32, True)
    q, k, qw, kw, cos, sin, pos, gq, gk = c

    def step():
        o = fused_qk_norm_rope(q, k, qw, kw, cos, sin, pos)
        return [t.detach() for t in o] + list(torch.autograd.grad(o, [q, k, qw, kw], (gq, gk)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _check_case(c, 1e-6, False)
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(3):
        with torch.no_grad():
            q.add_(0.1 * i)
            k.mul_(1 - 0.05 * i)
        graph.replay()
        got = [o.clone() for o in outs]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.gpu
def test_gpu_no_second_derivative():
    q, k, qw, kw, cos, sin, pos, gq, _ = _case("cuda", (4,), 2, 1, 32, 16, False, torch.float32, torch.float32, False)
    qo, _ = fused_qk_norm_rope(q, k, qw, kw, cos, sin, pos)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(qo, q, gq, create_graph=True)


def _frozen(dev):
    g = torch.Generator().manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g).to(dev)
    q, k, qw, kw, gq, gk = rnd(2, 9, 4, 24), rnd(2, 9, 2, 24), rnd(24), rnd(24), rnd(2, 9, 4, 24), rnd(2, 9, 2, 24)
    pos = torch.arange(9, device=dev)
    tables = rotary_tables(16, 16, device=dev)
    given = [t.requires_grad_(True) for t in (q, k, qw, kw)]
    for weights in (True, False):
        leaves = given if weights else given[:2]
        pick = lambda ts: list(ts) if weights else list(ts[:2]) + [None, None]
        full = torch.autograd.grad(fused_qk_norm_rope(*pick(given), *tables, pos), leaves, (gq, gk))
        for t, want in zip(leaves, full):
            only = pick([v if v is t else v.detach() for v in given])
            outs = fused_qk_norm_rope(*only, *tables, pos)
            pairs = [(o, go) for o, go in zip(outs, (gq, gk)) if o.requires_grad]
            got, = torch.autograd.grad([o for o, _ in pairs], t, [go for _, go in pairs])
            assert torch.equal(got, want)
    # one output alone: the other's input takes no gradient from it
    qo, _ = fused_qk_norm_rope(*given, *tables, pos)
    dq, dk = torch.autograd.grad(qo, [q, k], gq, allow_unused=True)
    want, = torch.autograd.grad(fused_qk_norm_rope(*given, *tables, pos), [q], (gq, gk))
    assert torch.equal(dq, want) and (dk is None or (dk == 0).all())


def test_cpu_frozen_leaves():
    _frozen("cpu")


@pytest.mark.gpu
def test_gpu_frozen_leaves():
    _frozen("cuda")


def _weight_layouts(dev):
    # weights of d entries in any shape, the head size among the head counts: each entry belongs to its element
    q, k, qw, kw, cos, sin, pos, gq, gk = _case(dev, (3,), 4, 4, 4, 4, False, torch.float32, torch.float32, False)
    leaves = [q, k, qw, kw]
    want = fused_qk_norm_rope(q, k, qw, kw, cos, sin, pos)
    want_g = torch.autograd.grad(want, leaves, (gq, gk))
    for shape in ((1, 4), (4, 1), (2, 2)):
        got = fused_qk_norm_rope(q, k, qw.view(shape), kw.view(shape), cos, sin, pos)
        got_g = torch.autograd.grad(got, leaves, (gq, gk))
        assert all(torch.equal(a, b) for a, b in zip(got + got_g, want + want_g))


def test_cpu_weight_layouts():
    _weight_layouts("cpu")


@pytest.mark.gpu
def test_gpu_weight_layouts():
    _weight_layouts("cuda")


# Tokens enough that every lane takes several heads (2048 blocks of 4 (64 / G) groups, G lanes a head, two heads a
# forward group), odd head counts (a group's second head past the last); half-split pairs: groups of 6, 5, 5, 32,
# 12, 64 and 64 lanes
LOOPED = [(14500, 80, 34), (17400, 72, 72), (17400, 72, 40), (2900, 512, 512), (7300, 24, 8), (1500, 200, 8), (1500, 400, 398)]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,d,rot", LOOPED)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                          (torch.float16, torch.float16), (torch.bfloat16, None)])
def test_gpu_more_heads_than_groups(tokens, d, rot, inter, dtype, wdtype):
    _check_case(_case("cuda", (tokens,), 7, 3, d, rot, inter, dtype, wdtype, True), 1e-6, inter)
