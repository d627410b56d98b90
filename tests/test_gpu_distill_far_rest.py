"""distill_top_logits, tail "bucket", where the student's classes that are not
kept are far below its kept ones: their gradient is r times their distribution
among themselves, whatever lies between."""
import pytest
import torch

from cign_b200.distill import distill_top_logits
from tests.class_rows import DTYPES, U, check, sum_ulps
from tests.test_gpu_distill import INF, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("temp", [0.05, 1.0, 30.0])
@pytest.mark.parametrize("c", [6, 60, 900, 30000])
def test_rest_far_below(cuda, c, temp, dtype):
    k = 3
    x, v, i, gen = make(cuda, 6, c, k, torch.float32, "bucket", temp)
    kept = torch.zeros(6, c, dtype=torch.bool, device=cuda).scatter_(1, i, True)
    gap = torch.tensor([[45.0], [200.0], [3000.0], [1e4], [0.0], [0.0]], device=cuda)
    x = torch.where(kept, x, x - gap).to(dtype)
    x[4] = torch.where(kept[4], x[4], torch.full_like(x[4], torch.finfo(dtype).min))   # a mask: all of the rest alike
    x[5] = torch.where(kept[5], x[5], torch.full_like(x[5], -1e4 if dtype != torch.float32 else -1e9))
    x.requires_grad_()
    v = v - 0.5
    g = 0.5 + torch.rand(6, generator=gen, device=cuda)
    z, q = x.detach().double() / temp, v.double().exp()
    m, m_rest = z.amax(1, keepdim=True), z.masked_fill(kept, -INF).amax(1, keepdim=True)
    s_rest = torch.where(kept, 0.0, (z - m_rest).exp()).sum(1, keepdim=True)
    share = torch.where(kept, 0.0, (z - m_rest).exp()) / s_rest
    logs = (z - m).exp().sum(1, keepdim=True).log()
    p, log_rest = (z - m - logs).exp(), (m_rest - m) + s_rest.log() - logs
    mass = q.sum(1, keepdim=True)
    r = 1 - mass
    target = torch.zeros_like(p).scatter_(1, i, q)
    kl = (q * (v.double() - (z - m - logs).gather(1, i))).sum(1, keepdim=True) + r * (r.log() - log_rest)
    want = temp ** 2 * kl[:, 0]
    want = torch.where(want > torch.finfo(torch.float32).max, INF, want)  # r T times the lowest value
    wgrad = (p - target - r * share) * temp * g.double()[:, None]
    ku = 2 * (sum_ulps(c) + 16) * U
    # the share: roundings of the rest's sum and of each exponent, relative to the rest's own maximum; kept classes as
    # differences of p and q, each with the roundings of its logarithm
    d_rest, d = torch.where(kept, 0.0, m_rest - z), torch.where(kept, m - z, 0.0)
    away = (p - target).abs() + target
    room = temp * g.double()[:, None] * (ku * (1 + d_rest + (share * d_rest).sum(1, keepdim=True)) * r * share
                                         + ku * (1 + d + d.sum(1, keepdim=True)) * (away + p) + 2.0 ** -125)
    loss = distill_top_logits(x, v, i, temp, "bucket")
    check(loss, want, temp ** 2 * ku * (1 + kl[:, 0].abs() + d.sum(1)), f"loss c={c} T={temp}")
    (grad,) = torch.autograd.grad(loss, x, g)
    check(grad, wgrad, room, f"grad c={c} T={temp}")
