"""Top-logit distillation loss against its definition in 64 bits.

Tolerances.  Gradient: one rounding to the logits' type (eps/2 of the value), plus the fp32 arithmetic:
1/T is folded into a base-2 scale (exponents up to 64 rounded to 2^-24 of themselves: 64 * 2^-24 * ln 2
relative error of each probability) and a sum of v terms in lanes of at most v/256 + 14 sequential
additions, 2^-24 each.  All of it stays below 2^-16 of a probability and of a teacher weight for
the vocabularies here.  Loss: the same error on the log terms, 2^-17 of the sum of the terms' magnitudes
plus eps/2 of its type, plus the logarithm of the sum: a relative error of (v/256 + 16) 2^-24 of a sum is
that absolute error of its logarithm however small the logarithm is, it enters every term with
weight t_k (sum 1) and the factor T^2."""
import pytest
import torch

from apex.contrib.xentropy import SoftmaxTopKDistillationLoss


def _exact(logits, tz, ti, temp, g=None):
    x = logits.detach().double()
    # the maximum goes first: a row at its type's lowest value would swallow the logarithm of the sum
    x = (x - x.amax(-1, keepdim=True)) / temp
    live = ti >= 0
    z = (tz.double() / temp).masked_fill(~live, float("-inf"))
    some = (z > float("-inf")).any(-1, keepdim=True)
    zz = torch.where(some, z, torch.zeros_like(z))
    t = torch.where(some & live, torch.softmax(zz, -1), torch.zeros_like(z))
    idx = ti.clamp(min=0).long()
    lq = (x - torch.logsumexp(x, -1, keepdim=True)).gather(1, idx)
    lt = torch.log_softmax(zz, -1)
    pos = t > 0
    terms = torch.where(pos, t * (torch.where(pos, lt, torch.zeros_like(t)) - lq), torch.zeros_like(t)) * temp ** 2
    mag = torch.where(pos, t * (torch.where(pos, lt, torch.zeros_like(t)).abs() + lq.abs()), torch.zeros_like(t))
    if g is None:
        return terms.sum(-1), mag.sum(-1) * temp ** 2
    q = torch.softmax(x, -1)
    tv = torch.zeros_like(q).scatter_add_(1, idx, t)
    s = (g.double() * temp)[:, None]
    some = some.to(q.dtype)
    return terms.sum(-1), mag.sum(-1) * temp ** 2, s * some * (q - tv), s.abs() * some * (q + tv)


def _case(dev, rows, v, top, dtype, seed=0, pitch=None, itype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    base = torch.randn(rows, v, generator=g)
    x = 3 * base + torch.randn(rows, v, generator=g)
    z, idx = (3 * base).topk(top, -1)
    if rows > 2:
        idx[1] = -1                      # no teacher
        idx[2, top // 2:] = -1           # fewer entries
    x = x.to(dtype).to(dev)
    if pitch is not None:                # rows of a padded buffer
        buf = torch.full((rows, pitch), float("nan"), dtype=dtype, device=dev)
        buf[:, :v] = x
        x = buf[:, :v]
    w = torch.rand(rows, generator=g).to(dev) + 0.5
    return x.detach().requires_grad_(True), z.to(dev), idx.to(itype).to(dev), w


def _check(x, z, idx, w, temp):
    loss = SoftmaxTopKDistillationLoss.apply(x, z, idx, temp, True)
    assert loss.dtype == torch.promote_types(x.dtype, torch.float32) and loss.shape == (x.size(0),)
    grad, = torch.autograd.grad(loss, x, w)
    assert grad.dtype == x.dtype and grad.shape == x.shape
    want, mag, dx, dmag = _exact(x, z, idx, temp, w)
    log_sum = temp ** 2 * (x.size(1) / 256 + 16) * 2.0 ** -24
    assert ((loss.double() - want).abs() <= 2.0 ** -17 * mag + 2.0 ** -24 * want.abs() + log_sum).all(), "loss"
    eps = torch.finfo(x.dtype).eps
    tiny = 2.0 ** -24 if x.dtype == torch.float16 else 2.0 ** -126
    err = (grad.double() - dx).abs()
    assert (err <= eps / 2 * 1.01 * dx.abs() + 2.0 ** -16 * dmag + tiny).all(), "gradient"
    empty = ((idx < 0) | (z == float("-inf"))).all(-1)
    assert (loss[empty] == 0).all() and (grad[empty] == 0).all()
    half = SoftmaxTopKDistillationLoss.apply(x, z, idx, temp)
    assert half.dtype == x.dtype and torch.equal(half, loss.to(x.dtype))


SHAPES = [(1, 1, 1), (3, 7, 3), (5, 8, 8), (4, 1000, 17), (3, 2049, 1), (2, 4103, 64)]


@pytest.mark.parametrize("rows,v,top", SHAPES)
@pytest.mark.parametrize("temp", [1.0, 2.5])
def test_cpu_loss(rows, v, top, temp):
    for dtype in (torch.float32, torch.bfloat16):
        _check(*_case("cpu", rows, v, top, dtype), temp)


def test_cpu_gradient_against_differences():
    x, z, idx, _ = _case("cpu", 4, 9, 3, torch.float64)
    idx[3] = torch.tensor([2, 5, 2])  # one class twice
    f = lambda x: SoftmaxTopKDistillationLoss.apply(x, z.double(), idx, 1.7, True)
    assert torch.autograd.gradcheck(f, (x,))


def _edges(dev, v=5003, dtype=torch.float32):
    inf = float("inf")
    x, z, idx, w = _case(dev, 9, v, 6, dtype)
    with torch.no_grad():
        x[1] = float("nan")              # a padding row may hold anything
        x[3, 100:] = -inf                # masked classes, none of the teacher's
        idx[3] = torch.arange(6, device=dev)
        x[4] = torch.finfo(dtype).min    # every class at the type's lowest value
        z[5, 2:] = -inf                  # entries of zero probability
        z[6] = -inf                      # ... and a row of them
        idx[7, 3] = idx[7, 0]            # one class twice
        idx[7, 5] = idx[7, 0]
    w[1] = float("nan")
    loss = SoftmaxTopKDistillationLoss.apply(x, z, idx, 2.0, True)
    grad, = torch.autograd.grad(loss, x, w)
    assert loss[1] == 0 and (grad[1] == 0).all() and loss[6] == 0 and (grad[6] == 0).all()
    keep = torch.tensor([0, 2, 3, 4, 5, 6, 7, 8], device=dev)
    with torch.no_grad():
        xs = x[keep].clone().requires_grad_(True)
    _check(xs, z[keep], idx[keep], w[keep], 2.0)
    # the teacher names a class that the student excludes: an infinite loss, a finite gradient
    with torch.no_grad():
        x[0, idx[0, 0]] = -inf
        x[8, 0] = float("nan")
    bad = idx.clone()
    bad[2, 0] = v                        # past the vocabulary
    loss = SoftmaxTopKDistillationLoss.apply(x, z, bad, 2.0, True)
    grad, = torch.autograd.grad(loss, x, torch.ones_like(w))
    assert loss[0] == inf and grad[0].isfinite().all()
    assert loss[2].isnan() and grad[2].isnan().all()
    assert loss[8].isnan() and loss[[3, 4, 5, 6, 7]].isfinite().all()


def test_cpu_edges():
    _edges("cpu")


def _refusals(dev):
    f = SoftmaxTopKDistillationLoss.apply
    x, z, i = torch.zeros(3, 9, device=dev), torch.zeros(3, 2, device=dev), torch.zeros(3, 2, dtype=torch.int64, device=dev)
    f(x, z, i)
    for err, args in [(ValueError, (x[0], z, i)), (ValueError, (x[:, :0], z, i)), (ValueError, (x, z[:2], i[:2])),
                      (ValueError, (x, z, i[:, :1])), (TypeError, (x, z, i.float())), (TypeError, (x, z.long(), i)),
                      (ValueError, (x, z, i, 0.0)), (ValueError, (x, z, i, -1.0)), (ValueError, (x, z, i, float("nan"))),
                      (ValueError, (x.long(), z, i)), (ValueError, (x, z.clone().requires_grad_(True), i))]:
        with pytest.raises(err):
            f(*args)


def test_cpu_refusals():
    _refusals("cpu")


def _temperature_range(dev):
    """1 / T or T^2 past fp32's range would make every loss NaN: refused; inside, the limits T -> 0 and T -> inf
    hold: one-hot distributions that agree, and terms of size 1 / T that vanish next to their coefficient."""
    f = SoftmaxTopKDistillationLoss.apply
    x = torch.tensor([[0.0, 3.0, 1.0, -2.0]], device=dev, requires_grad=True)
    z, i = torch.tensor([[2.0, 1.0]], device=dev), torch.tensor([[1, 2]], device=dev)
    for t in (1e-46, 1e-16, 1e16, 1e39, 1e-320):
        with pytest.raises(ValueError):
            f(x, z, i, t)
    loss = f(x, z, i, 1e-15, True)
    grad, = torch.autograd.grad(loss.sum(), x)
    assert loss.item() == 0 and (grad == 0).all()
    assert torch.isfinite(f(x, z, i, 1e15, True)).all()


def test_cpu_temperature_range():
    _temperature_range("cpu")


# ------------------------------------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("rows,v,top", SHAPES + [(2, 50257, 33), (1100, 3001, 5), (1, 131072, 1024), (1025, 257, 256)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("temp", [0.5, 1.0, 2.5])
def test_gpu_loss(rows, v, top, dtype, temp):
    _check(*_case("cuda", rows, v, top, dtype), temp)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gpu_row_pitch_index_type_and_order(dtype):
    x, z, idx, w = _case("cuda", 37, 5001, 20, dtype, pitch=5024, itype=torch.int32)
    _check(x, z, idx, w, 2.0)
    _check(x, z.to(torch.bfloat16).float().to(torch.bfloat16), idx, w, 2.0)  # teacher logits of 16 bits
    perm = torch.randperm(20, device="cuda")
    _check(x, z[:, perm].t().contiguous().t(), idx[:, perm], w, 2.0)        # unsorted, transposed storage
    xt = x.detach().t().contiguous().t().requires_grad_(True)                # classes not contiguous
    _check(xt, z, idx, w, 2.0)


@pytest.mark.gpu
@pytest.mark.parametrize("v", [200, 5003, 70001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gpu_edges(v, dtype):
    _edges("cuda", v, dtype)


@pytest.mark.gpu
def test_gpu_refusals():
    _refusals("cuda")
    f = SoftmaxTopKDistillationLoss.apply
    x = torch.zeros(3, 2000, device="cuda")
    i = torch.zeros(3, 1025, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError):
        f(x, i.float(), i)
    with pytest.raises(ValueError):
        f(x, i[:, :2].float(), i[:, :2].cpu())
    with pytest.raises(TypeError):
        f(x.double(), i[:, :2].float(), i[:, :2])


@pytest.mark.gpu
def test_gpu_temperature_range():
    _temperature_range("cuda")


@pytest.mark.gpu
def test_gpu_empty_rows_entries_and_broadcast_gradient():
    f = SoftmaxTopKDistillationLoss.apply
    x = torch.randn(4, 100, device="cuda", requires_grad=True)
    none = torch.zeros(4, 0, device="cuda")
    loss = f(x, none, none.long(), 1.0, True)
    assert (loss == 0).all()
    loss.sum().backward()
    assert (x.grad == 0).all()
    e = torch.randn(0, 100, device="cuda", requires_grad=True)
    f(e, none[:0], none[:0].long()).sum().backward()
    assert e.grad.shape == (0, 100)
    x, z, idx, _ = _case("cuda", 64, 777, 9, torch.float32)
    a, = torch.autograd.grad(f(x, z, idx, 1.0, True).sum(), x)  # a stride-0 gradient
    b, = torch.autograd.grad(f(x, z, idx, 1.0, True), x, torch.ones(64, device="cuda"))
    assert torch.equal(a, b)


@pytest.mark.gpu
def test_gpu_offsets_past_32_bits():
    rows, v = 9, 1 << 28  # 9 * 2^28 elements: the last rows start past 2^31
    x = torch.zeros(rows, v, dtype=torch.bfloat16, device="cuda")
    x[-1, -1] = 20.0
    z = torch.zeros(rows, 1, device="cuda")
    idx = torch.full((rows, 1), v - 1, device="cuda")
    x.requires_grad_(True)
    loss = SoftmaxTopKDistillationLoss.apply(x, z, idx, 1.0, True)
    want = torch.full((rows,), v, dtype=torch.float64).log()
    want[-1] = torch.log(torch.tensor(v - 1.0, dtype=torch.float64) + torch.tensor(20.0, dtype=torch.float64).exp()) - 20
    torch.testing.assert_close(loss.cpu().double(), want, rtol=1e-5, atol=0)
    grad, = torch.autograd.grad(loss, x, torch.ones_like(loss))
    q = (20.0 - want[-1].item() - 20.0)
    assert abs(grad[-1, -1].item() - (torch.tensor(q).exp().item() - 1)) < 2 ** -8
    assert grad[0, -1].item() == -1.0 and grad[-1, 0].item() > 0


@pytest.mark.gpu
def test_gpu_other_stream_captured_graph_and_repeatability():
    x, z, idx, w = _case("cuda", 40, 30011, 21, torch.bfloat16)

    def step():
        loss = SoftmaxTopKDistillationLoss.apply(x, z, idx, 2.0, True)
        return loss.detach(), torch.autograd.grad(loss, x, w)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _check(x, z, idx, w, 2.0)
        step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(step(), step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(3):
        with torch.no_grad():
            x.mul_(1 - 0.1 * i)
            idx.copy_(torch.where(idx >= 0, (idx + i) % 30011, idx))
        graph.replay()
        got = [o.clone() for o in outs]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.gpu
def test_gpu_no_second_derivative():
    x, z, idx, w = _case("cuda", 5, 99, 4, torch.float32)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(SoftmaxTopKDistillationLoss.apply(x, z, idx, 1.0, True), x, w, create_graph=True)


@pytest.mark.gpu
def test_gpu_more_rows_than_a_launch_has():
    # 512 threads a row: 2^32 threads are 2^23 rows.  Rows on both sides of it against 64 bits.
    rows, v = (1 << 23) + 5, 3
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(rows, v, device="cuda", generator=g).to(torch.bfloat16).requires_grad_(True)
    z = torch.randn(rows, 2, device="cuda", generator=g)
    idx = torch.tensor([2, 0], dtype=torch.int32, device="cuda").repeat(rows, 1)
    idx[-1] = -1
    w = torch.rand(rows, device="cuda", generator=g)
    _check(x, z, idx, w, 2.0)


def _lowest_values(dev, dtype, temp):
    """Logits at the lowest value of their type, the student's or the teacher's: x / T is no fp32 number there
    below T = 1, and log q (up to 3.4e38 / T) overflows where T^2 t log q does not."""
    low = torch.finfo(torch.float32).min
    x = torch.tensor([[0.0, 1.0, 2.0, -1.0, 0.5]], device=dev).repeat(5, 1).to(dtype)
    x[0] = torch.finfo(dtype).min                 # every class
    x[1, 2:] = torch.finfo(dtype).min             # masked ones, none of the teacher's
    x[3, 0] = torch.finfo(dtype).min              # one that the teacher names
    z = torch.tensor([[0.5, 0.5]], device=dev).repeat(5, 1)
    z[2] = low                                    # a teacher that knows no difference
    z[4, 0] = low                                 # ... and one that excludes an entry
    idx = torch.tensor([[0, 1]], device=dev).repeat(5, 1)
    w = torch.tensor([0.5, 0.75, 1.0, 1.25, 1.5], device=dev)
    _check(x.requires_grad_(True), z, idx, w, temp)


@pytest.mark.parametrize("temp", [0.25, 1.0, 1.5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_cpu_lowest_values(dtype, temp):
    _lowest_values("cpu", dtype, temp)


@pytest.mark.gpu
@pytest.mark.parametrize("temp", [0.25, 1.0, 1.5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_gpu_lowest_values(dtype, temp):
    _lowest_values("cuda", dtype, temp)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_gpu_streamed_logits(dtype):
    # past 256 MiB the forward streams the logits; an odd vocabulary, so that rows start inside vectors
    v, top = 131073, 16
    rows = (260 << 20) // (v * torch.finfo(dtype).bits // 8) + 1
    g = torch.Generator(device="cuda").manual_seed(11)
    x = (3 * torch.randn(rows, v, device="cuda", generator=g)).to(dtype)
    idx = torch.randint(0, v, (rows, top), device="cuda", generator=g)
    idx[:, 0], idx[:, 1] = v - 1, 0               # the row's ends
    z = 3 * torch.randn(rows, top, device="cuda", generator=g)
    w = torch.rand(rows, device="cuda", generator=g) + 0.5
    loss = SoftmaxTopKDistillationLoss.apply(x.requires_grad_(True), z, idx, 2.0, True)
    grad, = torch.autograd.grad(loss, x, w)
    eps = torch.finfo(dtype).eps
    tiny = 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -126
    for r in range(0, rows, 100):                 # the bounds of _check, in blocks of rows
        b = slice(r, r + 100)
        want, mag, dx, dmag = _exact(x[b], z[b], idx[b], 2.0, w[b])
        log_sum = 2.0 ** 2 * (v / 256 + 16) * 2.0 ** -24
        assert ((loss[b].double() - want).abs() <= 2.0 ** -17 * mag + 2.0 ** -24 * want.abs() + log_sum).all()
        assert ((grad[b].double() - dx).abs() <= eps / 2 * 1.01 * dx.abs() + 2.0 ** -16 * dmag + tiny).all()
