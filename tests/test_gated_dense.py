"""Gated feed-forward block against its formulas in 64 bits.

Tolerances.  Let e = eps/2 of the type (one rounding).  A k-term product sum in MFMA steps errs by at most (k/16 + 16) 2^-24 of the sum of its terms' magnitudes.
h, da and du are rounded to the type between the products, so each output's error is bounded by the
64-bit sum of its terms' magnitudes, times the roundings its terms carry (one e each):
  y, dW2: h        dx, dW1, db1: da, du
The pre-activations kept for the backward are cut to 24 bits (2^-15 of a value): da, du change by at most
2^-15 of |dh| |u| (|act'| + |a| sup|act''|) and |dh| (|act| + |a| sup|act'|) (sup|act''| 0.5 for silu and 1.13
for gelu, sup|act'| 1.13).  Each output has one rounding (e) of its own."""
import math

import pytest
import torch

from apex.fused_dense import FusedDenseGatedDense, fused_dense_gated_dense_function


def _act(a, kind):
    if kind == "silu":
        s = torch.sigmoid(a)
        return a * s, s * (1 + a * (1 - s))
    c0, c1 = math.sqrt(2 / math.pi), 0.044715
    th = torch.tanh(c0 * (a + c1 * a ** 3))
    return 0.5 * a * (1 + th), 0.5 * (1 + th) + 0.5 * a * (1 - th * th) * c0 * (1 + 3 * c1 * a * a)


def _exact(x, w1, b1, w2, b2, kind, dy):
    """{name: (value, terms that carry a rounding, terms that carry the 24-bit cut, summed length, terms of the
    sums inside dh)} in 64 bits."""
    x, w1, w2, dy = (t.detach().double().cpu() for t in (x, w1, w2, dy))
    f = w2.size(1)
    au = x @ w1.t() + (0 if b1 is None else b1.detach().double().cpu())
    a, u = au[:, :f], au[:, f:]
    act, dact = _act(a, kind)
    h = act * u
    # an fp32 sum of k terms behind a and u enters everything after them; it is far below e of the type
    y = h @ w2.t() + (0 if b2 is None else b2.detach().double().cpu())
    dh = dy @ w2
    dau = torch.cat((dh * u * dact, dh * act), 1)
    dhm = dy.abs() @ w2.abs()
    # dh's own fp32 error is relative to dhm, the roundings of da and du to themselves
    cut = torch.cat((dh.abs() * u.abs() * (dact.abs() + 1.13 * a.abs()), dh.abs() * (act.abs() + 1.13 * a.abs())), 1)
    mag = dau.abs()
    sums = torch.cat((dhm * u.abs() * dact.abs(), dhm * act.abs()), 1)
    # an error of a's or u's fp32 sum reaches h by |u| sup|act'| and |act|
    hm = h.abs() + 1.13 * a.abs() * u.abs()
    m, k = x.shape
    n = w2.size(0)
    return {
        "y": (y, h.abs() @ w2.abs().t(), 0, f, hm @ w2.abs().t()),
        "dx": (dau @ w1, mag @ w1.abs(), cut @ w1.abs(), 2 * f, (sums + cut) @ w1.abs()),
        "dw1": (dau.t() @ x, mag.t() @ x.abs(), cut.t() @ x.abs(), m, (sums + cut).t() @ x.abs()),
        "db1": (dau.sum(0), mag.sum(0), cut.sum(0), m, (sums + cut).sum(0)),
        "dw2": (dy.t() @ h, dy.abs().t() @ h.abs(), 0, m, dy.abs().t() @ hm),
        "db2": (dy.sum(0), 0, 0, m, dy.abs().sum(0)),
    }


def _close(got, want, mag, cut, length, sums, k, what):
    e = torch.finfo(got.dtype).eps / 2
    f32 = 2.0 ** -24
    bound = 1.01 * e * (want.abs() + mag) + 2.0 ** -15 * cut + sums * (length / 16 + k / 16 + 48) * f32
    bound = bound + (2.0 ** -24 if got.dtype == torch.float16 else 0.0)
    # an fp16 h, da or du near zero is rounded in steps of 2^-24
    if got.dtype == torch.float16:
        bound = bound + length * 2.0 ** -24
    ratio = ((got.detach().double().cpu() - want).abs() / bound.clamp(min=1e-300)).max()
    assert got.isfinite().all() and ratio <= 1, f"{what}: {float(ratio):.3f} bounds"


def _inputs(dev, m, k, f, n, dtype, bias, seed=0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(dtype).to(dev)
    x, w1, w2 = rnd(m, k), rnd(2 * f, k, std=k ** -0.5), rnd(n, f, std=f ** -0.5)
    b1, b2 = (rnd(2 * f, std=0.3), rnd(n, std=0.3)) if bias else (None, None)
    for t in (x, w1, w2, b1, b2):
        if t is not None:
            t.requires_grad_(True)
    return x, w1, b1, w2, b2, rnd(m, n)


def _check(x, w1, b1, w2, b2, dy, kind):
    y = fused_dense_gated_dense_function(x, w1, b1, w2, b2, kind)
    leaves = dict(dx=x, dw1=w1, db1=b1, dw2=w2, db2=b2)
    leaves = {a: t for a, t in leaves.items() if t is not None}
    grads = torch.autograd.grad(y, list(leaves.values()), dy)
    want = _exact(x, w1, b1, w2, b2, kind, dy)
    k = max(x.size(1), w2.size(0))
    _close(y, *want["y"], k, "y")
    for name, g in zip(leaves, grads):
        _close(g, *want[name], k, name)
    with torch.no_grad():
        assert torch.equal(fused_dense_gated_dense_function(x, w1, b1, w2, b2, kind), y)


def test_cpu_block_and_module():
    for kind in ("silu", "gelu"):
        _check(*_inputs("cpu", 5, 12, 7, 9, torch.float32, True), kind)
        m = FusedDenseGatedDense(6, 10, 4, bias=True, activation=kind).double()
        x = torch.randn(2, 3, 6, dtype=torch.float64, requires_grad=True)
        assert torch.autograd.gradcheck(lambda x, *p: fused_dense_gated_dense_function(x, p[0], p[2], p[1], p[3], kind),
                                        (x, m.weight1, m.weight2, m.bias1, m.bias2))
        assert m(x).shape == (2, 3, 4) and FusedDenseGatedDense(6, 10, 4).bias1 is None


def _autocast(dev, dtype):
    m = FusedDenseGatedDense(16, 24, 8, bias=True).to(dev)
    x = torch.randn(5, 16, device=dev)
    with torch.autocast(dev, dtype=dtype):
        y = m(x)
    assert y.dtype == dtype
    y.float().sum().backward()
    assert all(p.grad.dtype == torch.float32 and p.grad.isfinite().all() for p in m.parameters())
    low = [p.detach().to(dtype) for p in (m.weight1, m.bias1, m.weight2, m.bias2)]
    assert torch.equal(y, fused_dense_gated_dense_function(x.to(dtype), *low))


def test_cpu_autocast():
    _autocast("cpu", torch.bfloat16)


@pytest.mark.gpu
def test_gpu_autocast():
    _autocast("cuda", torch.float16)


def _refusals(dev):
    f = fused_dense_gated_dense_function
    z = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device=dev)
    x, w1, w2 = z(3, 8), z(32, 8), z(8, 16)
    f(x, w1, None, w2, None)
    for err, args in [(ValueError, (x, w1, None, w2, None, "relu")), (ValueError, (x, z(31, 8), None, w2, None)),
                      (ValueError, (z(3, 9), w1, None, w2, None)), (ValueError, (x, w1, z(16), w2, None)),
                      (ValueError, (x, w1, None, w2, z(9))), (TypeError, (x, w1.half(), None, w2, None)),
                      (TypeError, (x, w1, z(32, dt=torch.bfloat16), w2, None)), (ValueError, (x, w1[0], None, w2, None)),
                      (ValueError, (x, z(0, 8), None, z(8, 0), None))]:
        with pytest.raises(err):
            f(*args)
    with pytest.raises(ValueError):
        FusedDenseGatedDense(4, 4, 4, activation="tanh")


def test_cpu_refusals():
    _refusals("cpu")


# ------------------------------------------------------------------------------------------- GPU
# one token; odd row counts around the tiles; widths that end inside a 16-byte k step, a 64-deep tile,
# a tile; splits over the tokens; several tiles each way
SHAPES = [(1, 8, 8, 8), (1, 256, 136, 64), (3, 64, 128, 72), (16, 104, 5504, 8), (17, 72, 264, 136), (24, 5512, 24, 16),
          (32, 264, 136, 520), (33, 512, 1000, 256), (64, 128, 64, 40),
          (65, 320, 520, 328), (127, 200, 344, 96), (257, 264, 712, 520), (700, 256, 384, 128), (2100, 136, 200, 72),
          (4097, 64, 72, 264)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,f,n", SHAPES)
@pytest.mark.parametrize("kind,bias", [("silu", False), ("gelu", True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gpu_block(m, k, f, n, kind, bias, dtype):
    _check(*_inputs("cuda", m, k, f, n, dtype, bias), kind)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,f,n", [(17, 16, 8200, 24), (32, 24, 11016, 40), (16, 8, 8200, 16)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gpu_few_rows_of_a_long_second_product(m, k, f, n, dtype):
    _check(*_inputs("cuda", m, k, f, n, dtype, True), "silu")


@pytest.mark.gpu
def test_gpu_layouts_and_leading_axes():
    x, w1, b1, w2, b2, dy = _inputs("cuda", 60, 64, 96, 48, torch.bfloat16, True)
    want = fused_dense_gated_dense_function(x, w1, b1, w2, b2)
    x3 = x.detach().view(3, 4, 5, 64)
    assert torch.equal(fused_dense_gated_dense_function(x3, w1, b1, w2, b2).view(60, 48), want)
    # transposed storage, rows of a wider buffer, a view that starts inside a 16-byte vector
    xt = x.detach().t().contiguous().t()
    wide = torch.randn(192, 72, device="cuda").to(torch.bfloat16)
    wide[:, 3:67] = w1.detach()
    flat = torch.zeros(48 * 96 + 1, device="cuda", dtype=torch.bfloat16)
    flat[1:] = w2.detach().reshape(-1)
    wv = flat[1:].view(48, 96)
    assert torch.equal(fused_dense_gated_dense_function(xt, wide[:, 3:67], b1, wv, b2), want)
    y = fused_dense_gated_dense_function(x, w1, b1, w2, b2)
    a = torch.autograd.grad(y, [x, w1, w2], dy, retain_graph=True)
    b = torch.autograd.grad(y, [x, w1, w2], dy.t().contiguous().t(), retain_graph=True)
    assert all(torch.equal(i, j) for i, j in zip(a, b))
    c = torch.autograd.grad(y.sum(), [w1])  # an expanded gradient, one leaf only
    d = torch.autograd.grad(fused_dense_gated_dense_function(x, w1, b1, w2, b2), [w1], torch.ones_like(dy))
    assert torch.equal(c[0], d[0])


@pytest.mark.gpu
@pytest.mark.parametrize("with1,with2", [(False, False), (True, False), (False, True), (True, True)])
def test_gpu_frozen_leaves(with1, with2):
    # either bias alone, and any single leaf that takes a gradient: the same bits as with all of them
    x, w1, b1, w2, b2, dy = _inputs("cuda", 70, 64, 96, 48, torch.bfloat16, True)
    b1, b2 = b1 if with1 else None, b2 if with2 else None
    given = [x, w1, b1, w2, b2]
    leaves = [t for t in given if t is not None]
    full = torch.autograd.grad(fused_dense_gated_dense_function(*given), leaves, dy)
    for t, want in zip(leaves, full):
        only = [v if v is t or v is None else v.detach() for v in given]
        y = fused_dense_gated_dense_function(*only)
        y.backward(dy)
        assert torch.equal(t.grad, want)


@pytest.mark.gpu
def test_gpu_no_tokens():
    x, w1, b1, w2, b2, _ = _inputs("cuda", 0, 64, 96, 48, torch.bfloat16, True)
    y = fused_dense_gated_dense_function(x, w1, b1, w2, b2)
    assert y.shape == (0, 48)
    y.sum().backward()
    assert x.grad.shape == (0, 64) and all((t.grad == 0).all() for t in (w1, b1, w2, b2))


@pytest.mark.gpu
def test_gpu_offsets_past_32_bits():
    # [tokens, 2 x intermediate] has 2.3e9 elements; its last rows against 64 bits
    x, w1, _, w2, _, _ = _inputs("cuda", 8, 64, 8192, 64, torch.bfloat16, False)
    m = 140000
    x = torch.randn(m, 64, device="cuda").to(torch.bfloat16).requires_grad_(True)
    dy = torch.randn(m, 64, device="cuda").to(torch.bfloat16)
    y = fused_dense_gated_dense_function(x, w1, None, w2, None)
    dx, = torch.autograd.grad(y, x, dy)
    tail = slice(m - 40, m)
    want = _exact(x[tail], w1, None, w2, None, "silu", dy[tail])
    _close(y[tail], *want["y"], 64, "y")
    _close(dx[tail], *want["dx"], 64, "dx")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_gpu_extreme_activations(kind):
    # gates far out on both sides: act and its derivative saturate, nothing overflows into NaN
    x = torch.eye(8, device="cuda", dtype=torch.bfloat16)
    vals = torch.tensor([-1e4, -200.0, -90.0, -20.0, 20.0, 90.0, 200.0, 1e4], device="cuda").to(torch.bfloat16)
    w1 = torch.cat((vals.expand(8, 8).t(), torch.ones(8, 8, device="cuda", dtype=torch.bfloat16))).contiguous()
    w2 = torch.eye(8, device="cuda", dtype=torch.bfloat16)
    w1.requires_grad_(True)
    y = fused_dense_gated_dense_function(x, w1, None, w2, None, kind)
    want, dwant = _act(vals.double(), kind)
    # fp32's exponential overflows past 88.7: a gate below that gives 0 for a value of at most 1e-36
    torch.testing.assert_close(y.detach().double(), want.expand(8, 8), rtol=1.01 * 2 ** -8, atol=1e-36)
    dw, = torch.autograd.grad(y, w1, torch.ones_like(y))
    torch.testing.assert_close(dw[:8].double(), dwant[:, None].expand(8, 8), rtol=2 ** -7, atol=1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [5, 40])
@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_gpu_square_of_a_pre_activation_past_fp32(kind, m):
    """a = -+2^67: act' is 0 and 1 there, though a^2 is no fp32 number.  Powers of two, each the single term of
    its sum: every value is exact."""
    x, w1, w2 = torch.zeros(m, 8), torch.zeros(16, 8), torch.zeros(8, 8)
    x[1, 0], x[2, 0], x[:, 1] = -2.0 ** 33, 2.0 ** 33, 1.0
    w1[0, 0], w1[8, 1], w2[0, 0] = 2.0 ** 34, 1.0, 1.0  # the first feature: a = 2^34 x0, u = 1
    x, w1, w2 = (t.to("cuda", torch.bfloat16).requires_grad_(True) for t in (x, w1, w2))
    y = fused_dense_gated_dense_function(x, w1, None, w2, None, kind)
    dy = torch.zeros_like(y)
    dy[1:3, 0] = 1.0
    dx, dw1, dw2 = torch.autograd.grad(y, (x, w1, w2), dy)
    want_y, want_dx, want_dw1, want_dw2 = torch.zeros(m, 8), torch.zeros(m, 8), torch.zeros(16, 8), torch.zeros(8, 8)
    want_y[2, 0] = 2.0 ** 67
    want_dx[2, 0], want_dx[2, 1] = 2.0 ** 34, 2.0 ** 67       # da = act'(a) u = 1, du = act(a)
    want_dw1[0, 0], want_dw1[0, 1] = 2.0 ** 33, 1.0           # da x of row 2
    want_dw1[8, 0], want_dw1[8, 1] = 2.0 ** 100, 2.0 ** 67    # du x
    want_dw2[0, 0] = 2.0 ** 67
    for got, want in ((y, want_y), (dx, want_dx), (dw1, want_dw1), (dw2, want_dw2)):
        assert torch.equal(got.detach().cpu().float(), want)


@pytest.mark.gpu
def test_gpu_nan_stays_in_its_row():
    x, w1, b1, w2, b2, dy = _inputs("cuda", 300, 72, 136, 64, torch.bfloat16, False)
    want = fused_dense_gated_dense_function(x, w1, None, w2, None).detach()
    with torch.no_grad():
        x[299] = float("nan")
        x[7, 3] = float("inf")
    y = fused_dense_gated_dense_function(x, w1, None, w2, None)
    keep = torch.ones(300, dtype=torch.bool, device="cuda")
    keep[[7, 299]] = False
    assert y[299].isnan().all() and torch.equal(y[keep], want[keep])


@pytest.mark.gpu
def test_gpu_refusals():
    _refusals("cuda")
    z = torch.zeros(32, 8, device="cuda")
    with pytest.raises(ValueError):
        fused_dense_gated_dense_function(z, z.cpu(), None, torch.zeros(8, 16), None)


@pytest.mark.gpu
def test_gpu_other_types_and_widths_run_the_torch_math():
    for dtype, shape in ((torch.float32, (9, 24, 40, 16)), (torch.bfloat16, (9, 23, 41, 15))):
        x, w1, b1, w2, b2, dy = _inputs("cuda", *shape, dtype, True)
        y = fused_dense_gated_dense_function(x, w1, b1, w2, b2)
        want = _exact(x, w1, b1, w2, b2, "silu", dy)["y"][0]
        torch.testing.assert_close(y.double().cpu(), want, rtol=0.02, atol=0.05 if dtype != torch.float32 else 1e-4)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [20, 1500])
def test_gpu_other_stream_captured_graph_and_repeatability(m):
    x, w1, b1, w2, b2, dy = _inputs("cuda", m, 128, 264, 192, torch.bfloat16, True)

    def step():
        y = fused_dense_gated_dense_function(x, w1, b1, w2, b2, "silu")
        return [y.detach()] + list(torch.autograd.grad(y, [x, w1, b1, w2, b2], dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _check(x, w1, b1, w2, b2, dy, "silu")
        step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(step(), step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(3):
        with torch.no_grad():
            x.mul_(1 - 0.1 * i)
            w2.add_(0.01 * i)
        graph.replay()
        got = [o.clone() for o in outs]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.gpu
def test_gpu_no_second_derivative():
    x, w1, b1, w2, b2, dy = _inputs("cuda", 5, 64, 72, 40, torch.bfloat16, False)
    y = fused_dense_gated_dense_function(x, w1, b1, w2, b2)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(y, x, dy, create_graph=True)


# Sizes whose products take the 256-wide tile, several K tiles deep and with ragged edges (SHAPES are 128-wide
# throughout): (tile width, splits of K) of gated, down, dW2, [da | du], dW1 and dx on 256 compute units
W, N = (256, 1), (128, 1)
PLANNED = [((777, 712, 4104, 264), [W, (128, 8), N, N, N, (128, 10)]),
           ((4099, 264, 520, 2056), [N, W, (128, 5), N, (128, 8), N]),
           ((523, 264, 4104, 2056), [N, (128, 5), W, N, N, (128, 15)]),
           ((4099, 264, 5512, 264), [W, (128, 5), (256, 5), N, N, (128, 5)]),
           ((4107, 520, 2056, 520), [N, (128, 3), (128, 5), W, (128, 3), (128, 3)]),
           ((523, 2600, 1544, 264), [N, (128, 3), N, N, W, (128, 4)]),
           ((4099, 2056, 520, 264), [N, N, (128, 8), N, (128, 3), W]),
           ((777, 2056, 5512, 264), [W, (128, 10), N, N, N, (256, 7)]),
           ((2057, 2600, 5512, 2056), [W, (256, 3), W, W, W, (256, 2)])]


def _plans(shape, cus):
    native = pytest.importorskip("apex._native")
    if not native.available():
        pytest.skip("native extension not built")
    return native.require("gated_ffn").gated_ffn.plans(*shape, cus)


@pytest.mark.parametrize("shape,plans", PLANNED)
def test_cpu_plans(shape, plans):
    """The sizes below stay on the kernels that they are there for."""
    assert _plans(shape, 256) == plans


@pytest.mark.gpu
@pytest.mark.parametrize("shape,plans", PLANNED)
@pytest.mark.parametrize("kind,bias,dtype", [("silu", True, torch.bfloat16), ("gelu", False, torch.bfloat16),
                                             ("silu", False, torch.float16), ("gelu", True, torch.float16)])
def test_gpu_wide_tiles(shape, plans, kind, bias, dtype):
    assert _plans(shape, torch.cuda.get_device_properties(0).multi_processor_count) == plans
    _check(*_inputs("cuda", *shape, dtype, bias), kind)


@pytest.mark.gpu
def test_gpu_autocast_bf16():
    _autocast("cuda", torch.bfloat16)


@pytest.mark.parametrize("shape", [(0, 64, 64, 64), (64, 0, 64, 64), (64, 64, 0, 64), (64, 64, 64, 1 << 30)])
def test_cpu_plans_of_no_product(shape):
    with pytest.raises(RuntimeError, match="out of range"):
        _plans(shape, 256)
