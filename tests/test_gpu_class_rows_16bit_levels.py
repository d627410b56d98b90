"""Gradients of 16-bit logits far from 0, in rows of more than 512 classes: an
exponent there is one operation on the logit, and what the rounding of its
constant part leaves must not reach the gradient.  Against 64 bits."""
import pytest
import torch

from cign_b200.distill import distill_top_logits
from cign_b200.node_log_probs import node_log_probs
from tests.class_rows import U, check, sum_ulps

pytestmark = pytest.mark.gpu


def logits(dev, c, level, dtype):
    """Eight rows around different levels, a few steps of the type between their values: probabilities of about
    1 / c and less, which float16 holds when the upstream gradient brings them near 1."""
    g = torch.Generator(device=dev).manual_seed(c)
    step = level * torch.finfo(dtype).eps
    at = level * (1 - 0.04 * torch.arange(8, device=dev).float())
    x = at[:, None] - step * torch.randint(0, 4, (8, c), generator=g, device=dev).float()
    return x.to(dtype).requires_grad_(), g


def exact(x, temp):
    z = x.detach().double() / temp
    logp = torch.log_softmax(z, 1)
    return z.amax(1, keepdim=True) - z, logp, logp.exp()


@pytest.mark.parametrize("dtype,level", [(torch.float16, 150.0), (torch.float16, 1500.0), (torch.float16, 5600.0),
                                         (torch.float16, -5600.0), (torch.bfloat16, 700.0), (torch.bfloat16, -5600.0)])
@pytest.mark.parametrize("c", [600, 901, 20000])
def test_log_prob_and_entropy_gradients(cuda, c, level, dtype):
    x, g = logits(cuda, c, level, dtype)
    d, logp, p = exact(x, 1.0)
    H = -torch.where(p > 0, p * logp, 0.0).sum(1, keepdim=True)
    labels = torch.zeros(8, dtype=torch.int64, device=cuda)
    gl = (0.25 * c) * (0.5 + torch.rand(8, generator=g, device=cuda))
    gh = gl * 0.1
    k = 2 * (sum_ulps(c) + 16) * U
    out = node_log_probs(x, labels)
    (a,) = torch.autograd.grad(out.log_prob, x, gl, retain_graph=True)
    (b,) = torch.autograd.grad((out.log_prob, out.entropy), x, (gl, gh))
    hit = torch.zeros_like(p)
    hit[:, 0] = 1.0
    G, GH = gl.double()[:, None], gh.double()[:, None]
    # the roundings of the row's sum, of the exponent (relative to itself) and of the products: no term in the level
    rel = k + 4 * U * (d + logp.abs())
    # an exponential below 2^-126, the smallest normal float32, is 0 (bf16 at 5600 has steps of 44: e^-88 and e^-131)
    none = 2.0 ** -125 * (G + GH * (1 + logp.abs().clamp(max=200.0) + H))
    lph = torch.where(p > 0, logp + H, 0.0)
    check(a, G * (hit - p), rel * G * (p + hit) + none, f"log_prob {level} c={c}")
    check(b, G * (hit - p) - GH * p * lph, rel * (G * (p + hit) + GH * p * (1 + logp.abs() + H)) + none,
          f"log_prob and entropy {level} c={c}")


@pytest.mark.parametrize("temp", [1.0, 3.0, 0.3])
@pytest.mark.parametrize("dtype,level", [(torch.float16, 150.0), (torch.float16, 1500.0), (torch.float16, -4000.0),
                                         (torch.bfloat16, 1500.0)])
@pytest.mark.parametrize("c", [600, 901, 20000])
def test_distillation_gradient(cuda, c, level, dtype, temp):
    x, g = logits(cuda, c, level * min(temp, 1.0), dtype)
    d, logp, p = exact(x, temp)
    values = torch.zeros(8, 2, device=cuda)
    index = torch.tensor([[0, 1]], device=cuda).expand(8, 2)
    gl = (0.25 * c / temp) * (0.5 + torch.rand(8, generator=g, device=cuda))
    (grad,) = torch.autograd.grad(distill_top_logits(x, values, index, temp, "drop"), x, gl)
    target = torch.zeros_like(p)
    target[:, :2] = 0.5
    k = 2 * (sum_ulps(c) + 16) * U
    G = temp * gl.double()[:, None]
    check(grad, G * (p - target), (k + 4 * U * (d + logp.abs())) * G * (p + target) + 2.0 ** -125 * G, f"{level} T={temp} c={c}")
