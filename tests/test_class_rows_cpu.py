"""Refusals of the class-row operators (layer_norm, node_log_probs,
distill_top_logits) that need no GPU: the C entry points check sizes, types and
pointers before anything is launched, the Python functions refuse CPU tensors."""
import ctypes

import pytest
import torch

from cign_b200 import _lib
from cign_b200.distill import distill_top_logits
from cign_b200.layer_norm import layer_norm
from cign_b200.node_log_probs import node_log_probs

INVALID, NULL, ALIGNMENT, UNSUPPORTED = 1, 2, 3, 6
P = ctypes.c_void_p(4096)  # stands for a device pointer: never followed, as every call below is refused


def ln_fwd(n=4, d=8, xt=0, pt=0, x=P, ldx=8, eps=1e-5, y=P, mean=None, rstd=None):
    return _lib.load_library().cign_layer_norm_fwd(n, d, xt, pt, x, ldx, None, None, eps, y, mean, rstd, None)


def ln_bwd(n=4, d=8, xt=0, pt=0, gy=P, ldg=8, x=P, ldx=8, mean=P, rstd=P, gx=P, gw=P, gb=P, ws=P, ws_bytes=1 << 30):
    return _lib.load_library().cign_layer_norm_bwd(n, d, xt, pt, gy, ldg, x, ldx, None, mean, rstd, gx, gw, gb, ws, ws_bytes, None)


def lp_fwd(n=4, c=8, xt=0, x=P, ld=8, labels=P, k=0, lp=P, ent=P, stats=P, top=None, idx=None):
    return _lib.load_library().cign_node_log_probs_fwd(n, c, xt, x, ld, labels, k, lp, ent, stats, top, idx, None)


def lp_bwd(n=4, c=8, xt=0, x=P, ld=8, labels=P, stats=P, ent=P, k=0, idx=None, gl=P, gh=P, gt=None, out=P):
    return _lib.load_library().cign_node_log_probs_bwd(n, c, xt, x, ld, labels, stats, ent, k, idx, gl, 1, gh, 1, gt, out, None)


def ds(back, n=4, c=8, xt=0, x=P, ld=8, k=2, vt=0, v=P, ldv=2, it=1, i=P, ldi=2, temp=1.0, tail=0, stats=P, loss=P, out=P):
    lib = _lib.load_library()
    args = (n, c, xt, x, ld, k, vt, v, ldv, it, i, ldi, temp, tail)
    return lib.cign_distill_bwd(*args, stats, loss, 1, out, None) if back else lib.cign_distill_fwd(*args, loss, stats, None)


@pytest.mark.parametrize("kw,code", [
    (dict(n=-1), INVALID), (dict(d=0), INVALID), (dict(xt=3), INVALID), (dict(pt=-1), INVALID), (dict(ldx=7), INVALID),
    (dict(eps=-1.0), INVALID), (dict(eps=float("nan")), INVALID), (dict(n=1 << 31), UNSUPPORTED),
    (dict(d=1 << 24, ldx=1 << 24), UNSUPPORTED), (dict(x=None), NULL), (dict(y=None), NULL), (dict(mean=P), NULL)])
def test_layer_norm_forward_refuses(kw, code):
    assert ln_fwd(**kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(n=-1), INVALID), (dict(d=-8), INVALID), (dict(xt=9), INVALID), (dict(ldx=7), INVALID), (dict(ldg=7), INVALID),
    (dict(gy=None), NULL), (dict(x=None), NULL), (dict(mean=None), NULL), (dict(rstd=None), NULL),
    (dict(ws=None), INVALID), (dict(ws_bytes=16), INVALID), (dict(ws=ctypes.c_void_p(4100)), ALIGNMENT)])
def test_layer_norm_backward_refuses(kw, code):
    assert ln_bwd(**kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(n=-1), INVALID), (dict(c=0), INVALID), (dict(xt=5), INVALID), (dict(ld=7), INVALID), (dict(k=9), INVALID),
    (dict(k=-1), INVALID), (dict(c=100, ld=100, k=65), UNSUPPORTED), (dict(c=1 << 31, ld=1 << 31), UNSUPPORTED),
    (dict(c=(1 << 31) - 1023, ld=1 << 31), UNSUPPORTED),
    (dict(x=None), NULL), (dict(labels=None), NULL), (dict(k=2), NULL), (dict(k=2, top=P), NULL),
    (dict(stats=ctypes.c_void_p(4100)), ALIGNMENT)])
def test_log_probs_forward_refuses(kw, code):
    assert lp_fwd(**kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(n=-1), INVALID), (dict(ld=3), INVALID), (dict(x=None), NULL), (dict(labels=None), NULL), (dict(stats=None), NULL),
    (dict(ent=None), NULL), (dict(out=None), NULL), (dict(k=2, gt=P), NULL), (dict(stats=ctypes.c_void_p(4100)), ALIGNMENT)])
def test_log_probs_backward_refuses(kw, code):
    assert lp_bwd(**kw) == code


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("kw,code", [
    (dict(n=-1), INVALID), (dict(c=0), INVALID), (dict(xt=4), INVALID), (dict(vt=4), INVALID), (dict(it=2), INVALID),
    (dict(ld=7), INVALID), (dict(k=0), INVALID), (dict(ldv=1), INVALID), (dict(ldi=1), INVALID), (dict(temp=0.0), INVALID),
    (dict(temp=float("nan")), INVALID), (dict(temp=float("inf")), INVALID), (dict(temp=1e-46), INVALID), (dict(tail=2), INVALID),
    (dict(k=257, ldv=257, ldi=257), UNSUPPORTED), (dict(c=(1 << 20) + 1, ld=1 << 21), UNSUPPORTED), (dict(x=None), NULL),
    (dict(v=None), NULL), (dict(i=None), NULL), (dict(loss=None), NULL), (dict(stats=ctypes.c_void_p(4104)), ALIGNMENT)])
def test_distill_refuses(back, kw, code):
    assert ds(back, **kw) == code


def test_distill_backward_needs_the_forwards_statistics():
    assert ds(True, stats=None) == NULL and ds(True, out=None) == NULL


def test_no_rows_launch_nothing():
    before = _lib.load_library().cign_kernel_launches()
    assert ln_fwd(n=0, x=None, y=None) == 0 and lp_fwd(n=0, x=None) == 0 and lp_bwd(n=0, x=None) == 0
    assert ds(False, n=0, x=None) == 0 and ds(True, n=0, x=None) == 0
    assert ln_bwd(n=0, gw=None, gb=None) == 0
    assert _lib.load_library().cign_kernel_launches() == before


def test_python_functions_refuse_cpu_tensors():
    x = torch.zeros(4, 8)
    with pytest.raises(TypeError):
        layer_norm(x)
    with pytest.raises(TypeError):
        node_log_probs(x, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(TypeError):
        distill_top_logits(x, torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int64))


def test_rows_of_copies_only_what_a_kernel_cannot_read():
    x = torch.zeros(4, 12)
    for t, ld, same in ((x, 12, True), (x[:, :5], 12, True), (x[:, 3:4], 12, True), (x[1:2], 12, True), (x[::2], 24, True),
                        (x.t(), 4, False), (x[:, ::2], 6, False), (x[:1].expand(4, 12), 12, False),
                        (x[:, :1].expand(4, 12), 12, False), (x[:0], 12, True)):
        rows, got = _lib.rows_of(t)
        assert got == ld and (rows.data_ptr() == t.data_ptr()) == same or t.numel() == 0
        assert rows.shape == t.shape


def test_classify_leaves_the_modes_of_the_parts(monkeypatch):
    """A part that was put in eval mode by itself stays so, after an error too."""
    from cign_b200 import model_cign
    model = model_cign.build_model(in_dim=8, hidden_dim=16, out_dim=3, num_layers=2, hop_scales=(1, 2), gat_heads=2)
    model.train()
    next(iter(model.children())).eval()
    modes = [m.training for m in model.modules()]
    assert True in modes and False in modes
    seen = []
    monkeypatch.setattr(model_cign.GraphCliffordNet, "forward",
                        lambda self, x, op: seen.append(any(m.training for m in self.modules())))
    monkeypatch.setattr(model_cign, "node_log_probs", lambda *a: "out")
    assert model.classify(None, None) == "out" and seen == [False]
    assert [m.training for m in model.modules()] == modes

    def fail(*a):
        raise ValueError("stop")
    monkeypatch.setattr(model_cign, "node_log_probs", fail)
    with pytest.raises(ValueError, match="stop"):
        model.classify(None, None)
    assert [m.training for m in model.modules()] == modes
