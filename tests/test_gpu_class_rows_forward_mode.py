"""A dual tensor (forward-mode differentiation) is refused by the class-row
operators, as by the framework's others: its tangent must not be lost."""
import pytest
import torch
from torch.autograd import forward_ad

from cign_b200.distill import distill_top_logits
from cign_b200.layer_norm import layer_norm
from cign_b200.node_log_probs import node_log_probs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(cuda, grad):
    x = torch.randn(5, 8, device=cuda)
    w = torch.randn(8, device=cuda)
    v, i = torch.zeros(5, 2, device=cuda), torch.tensor([[0, 1]], device=cuda).expand(5, 2)
    y = torch.zeros(5, dtype=torch.int64, device=cuda)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        plain = (layer_norm(x, w, w), node_log_probs(x, y, 2), distill_top_logits(x, v, i))
        xd = forward_ad.make_dual(x, torch.ones_like(x))
        wd = forward_ad.make_dual(w, torch.ones_like(w))
        vd = forward_ad.make_dual(v, torch.ones_like(v))
        xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()  # the autograd node's own refusal
        for call in (lambda: layer_norm(xd), lambda: layer_norm(xd, w, w), lambda: layer_norm(x, wd),
                     lambda: layer_norm(x, None, wd), lambda: node_log_probs(xd), lambda: node_log_probs(xd, y, 2),
                     lambda: layer_norm(xd, wg), lambda: layer_norm(xg, wd), lambda: distill_top_logits(xg, vd, i),
                     lambda: distill_top_logits(xd, v, i), lambda: distill_top_logits(x, vd, i)):
            with pytest.raises((RuntimeError, NotImplementedError, ValueError)):
                call()
    # a level that holds no dual tensor of the call changes nothing
    assert torch.equal(plain[0], layer_norm(x, w, w)) and torch.equal(plain[2], distill_top_logits(x, v, i))
    for a, b in zip(plain[1], node_log_probs(x, y, 2)):
        assert torch.equal(a, b)


def test_function_transforms_are_refused(cuda):
    x, v, i = torch.randn(5, 8, device=cuda), torch.zeros(5, 2, device=cuda), torch.tensor([[0, 1]], device=cuda).expand(5, 2)
    for f in (layer_norm, lambda t: node_log_probs(t).entropy, lambda t: distill_top_logits(t, v, i)):
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (x,), (torch.ones_like(x),))
        with pytest.raises(RuntimeError):
            torch.func.vmap(f)(x[None])
