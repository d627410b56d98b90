"""layer_norm of rows whose level is far above their spread, down to rows of one
value: the mean's own rounding must not reach the result.  Against 64 bits."""
import pytest
import torch

from cign_b200.layer_norm import layer_norm
from tests.class_rows import DTYPES, U, check, sum_ulps

pytestmark = pytest.mark.gpu
EPS = 1e-5
LEVELS = (12345.0, 1000.1, -54321.7, 0.1, 65000.0, -333.3)


def reference(x, w, b, gy, eps):
    """y and the gradients, and what their errors are measured by.  mu, the mean in float32, is off by dmu at most;
    e = x - mu is exact or rounded once.  Its mean <e> is off by the roundings k of a sum of values of its own size,
    |x - mean| + dmu, not of x's: that is dxh.  The variance <e^2> - <e>^2 is off by k roundings of <e^2>."""
    x, gy, w, b = (t.detach().double() for t in (x, gy, w, b))
    mean = x.mean(1, keepdim=True)
    e = x - mean
    e = e - e.mean(1, keepdim=True)  # the 64-bit mean's own rounding
    e = torch.where(e.abs() <= 1e-12 * x.abs(), 0.0, e)
    var = e.pow(2).mean(1, keepdim=True)
    rstd = (var + eps).rsqrt()
    xh, u = e * rstd, gy * w
    gx = rstd * (u - u.mean(1, keepdim=True) - xh * (u * xh).mean(1, keepdim=True))
    k = (sum_ulps(x.size(1)) + 8) * U
    dmu = k * x.abs().mean(1, keepdim=True)
    size = (e.abs() + dmu) * rstd                       # of e as it is formed, times rstd
    most = size.mean(1, keepdim=True)
    rel = k * (var + dmu.pow(2)) / (var + eps) + 4 * U  # of rstd
    dxh = k * most + 4 * U * size + rel * xh.abs()
    ua, uxa = u.abs().mean(1, keepdim=True), (u * xh).abs().mean(1, keepdim=True)
    # <u xh> as <u e> - <e> <u>, and its products with e and <e> apart
    duxh = (u.abs() * dxh).mean(1, keepdim=True) + k * ((u.abs() * size).mean(1, keepdim=True) + most * ua)
    tgx = rstd * (k * (u.abs() + ua) + (dxh + 4 * U * (size + most)) * (uxa + duxh) + xh.abs() * duxh) + rel * gx.abs()
    return dict(y=xh * w + b, ty=dxh * w.abs() + 2 * U * ((xh * w).abs() + b.abs()), gx=gx, tgx=tgx,
                gw=(gy * xh).sum(0), tgw=(gy.abs() * dxh).sum(0) + 90 * U * (gy * xh).abs().sum(0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("spread", ["none", "last digits", "small"])
@pytest.mark.parametrize("d", [3, 47, 96, 301, 520, 1000, 2560, 5003, 8192, 9000, 10080, 20000, 40001])
def test_level_far_above_the_spread(cuda, d, spread, dtype):
    g = torch.Generator(device=cuda).manual_seed(d)
    n = 13
    level = torch.tensor([LEVELS[r % len(LEVELS)] for r in range(n)], device=cuda).to(dtype)[:, None]
    x = level.expand(n, d).clone()
    if spread == "last digits":  # the level and its neighbour
        up = level.float().abs() * torch.finfo(dtype).eps
        x = torch.where(torch.rand(n, d, generator=g, device=cuda) < 0.3, (level.float() + up).to(dtype), x)
    elif spread == "small":
        x = (level.float() + 0.01 * torch.randn(n, d, generator=g, device=cuda)).to(dtype)
    assert torch.isfinite(x).all()
    x.requires_grad_()
    w = (1 + 0.1 * torch.randn(d, generator=g, device=cuda)).requires_grad_()
    b = (0.1 * torch.randn(d, generator=g, device=cuda)).requires_grad_()
    gy = torch.randn(n, d, generator=g, device=cuda).to(dtype)
    r = reference(x, w, b, gy, EPS)
    y = layer_norm(x, w, b, EPS)
    gx, gw = torch.autograd.grad(y, (x, w), gy)
    (gw_only,) = torch.autograd.grad(layer_norm(x.detach(), w, b, EPS), (w,), gy)
    what = f"d={d} {spread} {dtype}"
    check(y, r["y"], r["ty"], f"y {what}")
    check(gx, r["gx"], r["tgx"], f"grad x {what}")
    check(gw, r["gw"], r["tgw"], f"grad w {what}")
    check(gw_only, r["gw"], r["tgw"], f"grad w alone {what}")


@pytest.mark.parametrize("d", [47, 1000, 9000, 20000])
def test_rows_of_one_value_are_the_bias(cuda, d):
    """Every level up to 65000.  The mean is off by k roundings of it, e by as much, and <e> by k roundings of that;
    half a step of the mean alone (2^-9) would be 0.6 of y at eps = 1e-5."""
    g = torch.Generator(device=cuda).manual_seed(d)
    x = (torch.rand(500, 1, generator=g, device=cuda) * 65000.0).expand(500, d).contiguous()
    b = torch.randn(d, generator=g, device=cuda)
    room = ((sum_ulps(d) + 8) * U) ** 2 * 65000.0 / EPS ** 0.5
    assert room < 1e-3
    assert layer_norm(x, eps=EPS).abs().max() <= room
    assert (layer_norm(x, None, b, EPS) - b).abs().max() <= room + 8 * U


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d", [(41, 8), (5003, 37), (4001, 96), (77, 301), (1003, 520), (3001, 777), (601, 2560), (333, 5003),
                                 (99, 9000), (49, 16001), (31, 40000)])
def test_far_rows_leave_their_neighbours_alone(cuda, n, d, dtype):
    """Far rows among others, in one warp and one after the other in a block: the others are bit for bit what they
    are without them, and the far ones right."""
    g = torch.Generator(device=cuda).manual_seed(n)
    x = torch.randn(n, d, generator=g, device=cuda).to(dtype)
    far = torch.rand(n, generator=g, device=cuda) < 0.3
    far[0] = True
    y0_in = torch.where(far[:, None], (12345.0 + x.float()).to(dtype), x).requires_grad_()
    w = (1 + 0.1 * torch.randn(d, generator=g, device=cuda)).requires_grad_()
    gy = torch.randn(n, d, generator=g, device=cuda).to(dtype)
    x.requires_grad_()
    clean, mixed = layer_norm(x, w), layer_norm(y0_in, w)
    (gx_clean,) = torch.autograd.grad(clean, x, gy)
    gx, gw = torch.autograd.grad(mixed, (y0_in, w), gy)
    assert torch.equal(mixed[~far], clean[~far]) and torch.equal(gx[~far], gx_clean[~far])
    r = reference(y0_in[far], w, torch.zeros_like(w), gy[far], EPS)
    check(mixed[far], r["y"], r["ty"], f"y n={n} d={d} {dtype}")
    check(gx[far], r["gx"], r["tgx"], f"grad x n={n} d={d} {dtype}")
    z = y0_in.detach().double()
    e = z - z.mean(1, keepdim=True)
    xh = e * (e.pow(2).mean(1, keepdim=True) + EPS).rsqrt()
    gd = gy.double()
    k = (sum_ulps(d) + n / 64 + 90) * U
    # rows that are not far: the mean's roundings, k of a mean of at most twice the spread
    check(gw, (gd * xh).sum(0), k * (gd.abs() * (3 + xh.abs())).sum(0), f"grad w n={n} d={d} {dtype}")
