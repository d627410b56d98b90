"""layer_norm against the formula in 64 bits: outputs and gradients for every
type, widths from 1 to many thousands, layouts, missing parameters, rows
without variance, far means, empty input, other streams, graph capture."""
import pytest
import torch

from cign_b200.graph_step import GraphedStep
from cign_b200.layer_norm import layer_norm
from tests.class_rows import DTYPES, U, check, layout, sum_ulps

pytestmark = pytest.mark.gpu
EPS = 1e-5


def reference(x, w, b, gy, eps):
    """y, grad x, grad w, grad b and what their errors are measured by."""
    x, gy = x.detach().double(), gy.double()
    d = x.size(1)
    w = torch.ones(d, dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    b = torch.zeros_like(w) if b is None else b.detach().double()
    mean = x.mean(1, keepdim=True)
    var = (x - mean).pow(2).mean(1, keepdim=True)
    rstd = (var + eps).rsqrt()
    xh = (x - mean) * rstd
    u = gy * w
    gx = rstd * (u - u.mean(1, keepdim=True) - xh * (u * xh).mean(1, keepdim=True))
    # the mean is off by the roundings of its sum (dmu); the variance of differences from it by dmu^2
    # and by its own roundings, relative to itself
    k = sum_ulps(d) + 8
    dmu = k * U * x.abs().mean(1, keepdim=True) * rstd
    rel = dmu.pow(2) / 2 + k * U
    dxh = dmu + xh.abs() * (rel + 2 * U)
    ty = dxh * w.abs() + 2 * U * (xh.abs() * w.abs() + b.abs())
    ua = u.abs().mean(1, keepdim=True)
    uxa = (u * xh).abs().mean(1, keepdim=True)
    duxh = (u.abs() * dxh).mean(1, keepdim=True)
    tgx = rstd * (k * U * (u.abs() + ua + xh.abs() * uxa) + dxh * uxa + xh.abs() * duxh) + rel * gx.abs()
    return dict(y=xh * w + b, gx=gx, gw=(gy * xh).sum(0), gb=gy.sum(0), ty=ty, tgx=tgx,
                gwa=(gy * xh).abs().sum(0), gba=gy.abs().sum(0), gwd=(gy.abs() * dxh).sum(0))


def run_case(dev, n, d, dtype, pdtype, kind="plain", has_w=True, has_b=True, mean=0.3, eps=EPS):
    g = torch.Generator(device=dev).manual_seed(n * 7 + d)
    x = torch.randn(n, d, generator=g, device=dev) * (0.5 + torch.rand(n, 1, generator=g, device=dev)) + mean
    x = layout(x, dtype, kind).requires_grad_()
    w = (1 + 0.1 * torch.randn(d, generator=g, device=dev)).to(pdtype).requires_grad_() if has_w else None
    b = (0.1 * torch.randn(d, generator=g, device=dev)).to(pdtype).requires_grad_() if has_b else None
    gy = layout(torch.randn(n, d, generator=g, device=dev), dtype, kind)
    y = layer_norm(x, w, b, eps)
    assert y.dtype == dtype and y.shape == (n, d)
    leaves = [t for t in (x, w, b) if t is not None]
    grads = dict(zip([id(t) for t in leaves], torch.autograd.grad(y, leaves, gy)))
    r = reference(x, w, b, gy, eps)
    what = f"n={n} d={d} {dtype} {kind}"
    check(y, r["y"], r["ty"], f"y {what}")
    check(grads[id(x)], r["gx"], r["tgx"], f"grad x {what}")
    # rows are added in shares and the shares one after the other
    k = (n / 64 + 64 + 16) * U
    if has_w:
        check(grads[id(w)], r["gw"], k * r["gwa"] + r["gwd"], f"grad w {what}")
    if has_b:
        check(grads[id(b)], r["gb"], k * r["gba"], f"grad b {what}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d", [(1, 1), (3, 2), (5, 7), (64, 8), (300, 33), (129, 64), (1000, 100),
                                 (77, 256), (513, 301), (40, 512), (33, 1000), (200, 1024),
                                 (17, 1025), (65, 2048), (50, 2560), (9, 4096), (7, 5003),
                                 (4, 8192), (6, 10240), (3, 16385), (2, 40000), (1, 70001)])
def test_outputs_and_gradients(cuda, n, d, dtype):
    run_case(cuda, n, d, dtype, torch.float32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["padded", "shifted"])
@pytest.mark.parametrize("n,d", [(70, 5), (70, 96), (70, 512), (9, 2560), (5, 9000)])
def test_layouts(cuda, n, d, kind, dtype):
    run_case(cuda, n, d, dtype, dtype, kind)


@pytest.mark.parametrize("has_w,has_b", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("pdtype", [torch.float32, torch.bfloat16])
def test_missing_parameters(cuda, has_w, has_b, pdtype):
    run_case(cuda, 130, 520, torch.bfloat16, pdtype, has_w=has_w, has_b=has_b)
    run_case(cuda, 11, 4100, torch.bfloat16, pdtype, has_w=has_w, has_b=has_b)


@pytest.mark.parametrize("n,d", [(20000, 64), (5000, 520), (30001, 37)])
def test_many_rows(cuda, n, d):
    run_case(cuda, n, d, torch.float32, torch.float32)
    run_case(cuda, n, d, torch.bfloat16, torch.bfloat16)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d", [(1, 3), (2, 3), (17, 3), (40, 1), (33, 9), (5000, 13), (40007, 31), (9001, 301),
                                 (3000, 1027), (1501, 2049), (2111, 4111), (700, 8175)])
def test_odd_widths_over_many_rows(cuda, n, d, dtype):
    """Rows that start anywhere within 16 bytes, more than the device holds at once.  Equal rows need not come
    out bit for bit equal: where a row starts decides how its sum is grouped, and each grouping is within the
    allowed error of the exact row."""
    run_case(cuda, n, d, dtype, torch.float32)
    x = torch.randn(1, d, device=cuda).to(dtype).repeat(n, 1)
    r = reference(x[:1], None, None, torch.ones_like(x[:1]), EPS)
    check(layer_norm(x), r["y"].expand(n, d), r["ty"].expand(n, d), f"equal rows n={n} d={d} {dtype}")


def test_neighbours_and_ends_are_not_read_into_a_row(cuda):
    """NaN around the matrix and in every second row leaves the other rows as they are."""
    for dtype in DTYPES:
        for n, d in ((9, 5), (300, 37), (40, 1033), (20, 4099)):
            buf = torch.full((n * d + 32,), float("nan"), dtype=dtype, device=cuda)
            x = buf[16:16 + n * d].view(n, d)
            x.copy_(torch.randn(n, d, device=cuda))
            clean = layer_norm(x)
            assert torch.isfinite(clean).all()
            x[::2] = float("nan")
            y = layer_norm(x)
            assert torch.equal(y[1::2], clean[1::2]) and torch.isnan(y[::2]).all()
            xr = x.clone().requires_grad_()
            gy = torch.randn(n, d, device=cuda).to(dtype)
            (gx,) = torch.autograd.grad(layer_norm(xr), xr, gy)
            assert torch.isfinite(gx[1::2]).all()


@pytest.mark.parametrize("d", [64, 777, 2560, 20000])
def test_far_mean(cuda, d):
    """A mean a thousand times the spread: the variance is formed from differences."""
    run_case(cuda, 21, d, torch.float32, torch.float32, mean=1000.0)


@pytest.mark.parametrize("scale", [1e15, 1e-15])
@pytest.mark.parametrize("d", [64, 777, 2560, 9000, 20000])
def test_rows_of_far_magnitude(cuda, d, scale):
    """Rows whose rstd^3 is no float32 number."""
    x = (scale * torch.randn(21, d, device=cuda)).requires_grad_()
    gy = torch.randn(21, d, device=cuda)
    y = layer_norm(x, eps=0.0)
    (gx,) = torch.autograd.grad(y, x, gy)
    r = reference(x, None, None, gy, 0.0)
    check(y, r["y"], r["ty"], f"y d={d} {scale}")
    check(gx, r["gx"], r["tgx"], f"grad x d={d} {scale}")


@pytest.mark.parametrize("d", [8, 515, 6000])
def test_rows_without_variance(cuda, d):
    x = torch.full((5, d), 3.0, device=cuda).requires_grad_()
    w = torch.full((d,), 2.0, device=cuda)
    b = torch.full((d,), 0.5, device=cuda)
    y = layer_norm(x, w, b, EPS)
    assert torch.equal(y, torch.full_like(y, 0.5))
    gy = torch.randn(5, d, device=cuda)
    (gx,) = torch.autograd.grad(y, x, gy)
    u = gy.double() * 2
    e = (u - u.mean(1, keepdim=True)) / EPS ** 0.5
    check(gx, e, (sum_ulps(d) + 8) * U * (u.abs() + u.abs().mean(1, keepdim=True)) / EPS ** 0.5, "grad x")


def test_nan_and_infinity_stay_in_their_row(cuda):
    x = torch.randn(9, 700, device=cuda)
    x[2, 5] = float("nan")
    x[6, 699] = float("inf")
    y = layer_norm(x)
    bad = torch.isnan(y).any(1).cpu()
    assert bad.tolist() == [i in (2, 6) for i in range(9)]
    assert torch.isfinite(y[[0, 1, 3, 4, 5, 7, 8]]).all()


def test_empty_and_leading_dimensions(cuda):
    w = torch.ones(16, device=cuda, requires_grad=True)
    x = torch.zeros(0, 16, device=cuda, requires_grad=True)
    y = layer_norm(x, w, None)
    gx, gw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert y.shape == (0, 16) and gx.shape == (0, 16) and torch.equal(gw, torch.zeros_like(gw))
    x = torch.randn(3, 5, 16, device=cuda)
    assert torch.equal(layer_norm(x, w), layer_norm(x.view(15, 16), w).view(3, 5, 16))
    assert torch.equal(layer_norm(x[0, 0]), layer_norm(x[0, :1])[0])


@pytest.mark.parametrize("expand", ["rows", "all"])
def test_broadcast_gradient_and_input(cuda, expand):
    """An upstream gradient and an input whose rows are one row in memory."""
    x = torch.randn(1, 96, device=cuda).expand(50, 96).detach().requires_grad_()
    w = torch.ones(96, device=cuda, requires_grad=True)
    gy = torch.randn(1, 96, device=cuda).expand(50, 96) if expand == "rows" else \
        torch.randn(1, 1, device=cuda).expand(50, 96)
    got = torch.autograd.grad(layer_norm(x, w), (x, w), gy)
    xc = x.detach().clone().contiguous().requires_grad_()
    want = torch.autograd.grad(layer_norm(xc, w), (xc, w), gy.contiguous())
    for a, e in zip(got, want):
        assert torch.equal(a, e)


def test_gradient_against_differences(cuda):
    g = torch.Generator(device=cuda).manual_seed(4)
    x = torch.randn(6, 40, generator=g, device=cuda, requires_grad=True)
    w = torch.randn(40, generator=g, device=cuda, requires_grad=True)
    b = torch.randn(40, generator=g, device=cuda, requires_grad=True)
    gy = torch.randn(6, 40, generator=g, device=cuda)
    grads = torch.autograd.grad(layer_norm(x, w, b), (x, w, b), gy)
    h = 2.0 ** -5

    def loss(*t):
        return (layer_norm(*t).double() * gy.double()).sum().item()
    for i, (leaf, grad) in enumerate(zip((x, w, b), grads)):
        v = torch.randn(leaf.shape, generator=g, device=cuda)
        v = v / v.norm()
        args = [x.detach(), w.detach(), b.detach()]
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + h * v, args[i] - h * v
        diff = (loss(*up) - loss(*down)) / (2 * h)
        # a unit step: third derivatives of order |gy| |w|, and the outputs' roundings over h
        room = h * h * float(gy.norm() * w.norm()) / 6 + 16 * U * float((gy.abs() * 4).sum()) / h
        assert abs(diff - float((grad.double() * v.double()).sum())) <= room


def test_only_wanted_gradients(cuda):
    x = torch.randn(30, 72, device=cuda)
    w = torch.randn(72, device=cuda, requires_grad=True)
    b = torch.randn(72, device=cuda, requires_grad=True)
    gy = torch.randn(30, 72, device=cuda)
    gw, gb = torch.autograd.grad(layer_norm(x, w, b), (w, b), gy)
    xr = x.clone().requires_grad_()
    full = torch.autograd.grad(layer_norm(xr, w, b), (xr, w, b), gy)
    assert torch.equal(gw, full[1]) and torch.equal(gb, full[2])
    (gx,) = torch.autograd.grad(layer_norm(xr, w.detach(), b.detach()), xr, gy)
    assert torch.equal(gx, full[0])
    (gb_only,) = torch.autograd.grad(layer_norm(x, None, b), b, gy)
    assert torch.equal(gb_only, gb)


def test_repeats_bit_for_bit_and_second_stream(cuda):
    x = torch.randn(3001, 600, device=cuda, requires_grad=True)
    w = torch.randn(600, device=cuda, requires_grad=True)
    gy = torch.randn(3001, 600, device=cuda)

    def step():
        y = layer_norm(x, w)
        return (y.detach(), *torch.autograd.grad(y, (x, w), gy))
    one = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        two = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, e in zip(two, one):
        assert torch.equal(a, e)


def test_two_captured_graphs(cuda):
    """Two graphs of different sizes, replayed in turn, keep their own workspaces."""
    def make(n, d):
        x = torch.randn(n, d, device=cuda, requires_grad=True)
        w = torch.randn(d, device=cuda, requires_grad=True)
        gy = torch.randn(n, d, device=cuda)
        out = {}

        def step():
            y = layer_norm(x, w)
            out["g"] = torch.autograd.grad(y, (x, w), gy)
            return y.detach()
        eager = step().clone(), *[t.clone() for t in out["g"]]
        return GraphedStep(step, cuda, warmup=2), out, eager, x, w
    a, b = make(500, 320), make(64, 2560)
    for _ in range(3):
        for graph, out, eager, *_rest in (a, b, a):
            y = graph()
            torch.cuda.synchronize()
            for got, want in zip((y, *out["g"]), eager):
                assert torch.equal(got, want)
    graph, _out, eager, x, w = a
    with torch.no_grad():
        x.copy_(torch.randn_like(x))
        want = layer_norm(x, w)
    assert torch.equal(graph(), want) and not torch.equal(want, eager[0])


def test_second_derivative_is_refused(cuda):
    x = torch.randn(4, 8, device=cuda, requires_grad=True)
    (g,) = torch.autograd.grad(layer_norm(x).pow(2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_refusals(cuda):
    x = torch.randn(4, 8, device=cuda)
    w = torch.ones(8, device=cuda)
    for args, error in (((x.double(),), TypeError), ((x.cpu(),), TypeError), ((x, w[:7]), ValueError),
                        ((x, w.cpu()), TypeError), ((x, w.half()), TypeError),
                        ((x.half(), w, w.half()), TypeError), ((x, w, w, -1.0), ValueError),
                        ((x, w, w, float("nan")), ValueError), ((x[:, :0],), ValueError),
                        ((x[0, 0],), ValueError)):
        with pytest.raises(error):
            layer_norm(*args)
