"""_lib.refuse_tangents, which keeps the operators that leave the autograd node out
from losing a tangent."""
import pytest
import torch
from torch.autograd import forward_ad

from cign_b200 import _lib


def test_refuses_dual_tensors_alone():
    x, w = torch.randn(4), torch.randn(4, requires_grad=True)
    _lib.refuse_tangents("op", x, None, w)
    with forward_ad.dual_level():
        _lib.refuse_tangents("op", x, None, w)
        dual = forward_ad.make_dual(x, torch.ones(4))
        for args in ((dual,), (x, dual), (None, dual.reshape(2, 2))):
            with pytest.raises(NotImplementedError, match="op has no forward-mode derivative"):
                _lib.refuse_tangents("op", *args)
            with torch.no_grad(), pytest.raises(NotImplementedError):
                _lib.refuse_tangents("op", *args)
    _lib.refuse_tangents("op", x, w)
