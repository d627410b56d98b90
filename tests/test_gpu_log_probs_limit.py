"""node_log_probs at the largest number of classes, 2^31 - 1024, where positions in
a row are next to the end of 32 bits: a label and best classes at both ends of the
row, and the gradient there."""
import math

import pytest
import torch

from cign_b200.node_log_probs import node_log_probs

pytestmark = pytest.mark.gpu


def test_most_classes(cuda):
    c = 2 ** 31 - 1024
    g = torch.Generator(device=cuda).manual_seed(1)
    x = torch.empty(1, c, dtype=torch.bfloat16, device=cuda)
    x.normal_(generator=g)
    best = [c - 1, 0, c - 8, 2 ** 30 + 5, 7]
    for i, j in enumerate(best):
        x[0, j] = 30.0 - 2 * i
    x.requires_grad_()
    lse = 0.0
    for part in x.detach()[0].split(2 ** 26):
        lse += float(torch.exp(part.double() - 30.0).sum())
    lse = 30.0 + math.log(lse)
    out = node_log_probs(x, torch.tensor([c - 1], device=cuda), 5)
    # a thread's four chains add 2^18 terms each, one after the other
    room = 2.0 ** 18 * 2.0 ** -24
    assert out.top_index[0].tolist() == best
    assert abs(float(out.log_prob.detach()) - (30.0 - lse)) <= room
    want = torch.tensor([30.0 - 2 * i - lse for i in range(5)], device=cuda)
    assert float((out.top_log_probs.detach()[0] - want).abs().max()) <= room
    (grad,) = torch.autograd.grad(out.log_prob.sum(), x)
    for at in (slice(0, 4096), slice(2 ** 30 - 2048, 2 ** 30 + 2048), slice(c - 4096, c)):
        p = torch.exp(x.detach()[0, at].double() - lse)
        e = -p
        if at.stop == c:
            e[-1] += 1.0
        assert bool(((grad[0, at].double() - e).abs() <= 2.0 ** -8 * e.abs() + 2 * room * p).all())
