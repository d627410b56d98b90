"""The classification head in use: the model's node_loss and classify on labels
and on a teacher's kept classes, against torch on the same logits; a captured
training step with distillation against eager ones; and layer_norm, a linear
classifier, node_log_probs and distill_top_logits one after the other against
the same chain in 64 bits."""
import copy

import pytest
import torch
import torch.nn.functional as F

from cign_b200 import synth
from cign_b200.distill import distill_top_logits
from cign_b200.graph_operator import (build_sparse_normalized_adjacency, prepare_fixed_csr_operator,
                                      prepare_gat_edge_index, to_graph_format)
from cign_b200.graph_step import GraphedStep
from cign_b200.layer_norm import layer_norm
from cign_b200.model_cign import build_model
from cign_b200.multihop_csr_pipeline import prepare_multihop_csr_operator
from cign_b200.node_log_probs import node_log_probs
from tests.class_rows import U
from tests.helpers import assert_parity

pytestmark = pytest.mark.gpu


def setup(dev, hidden=64, layers=2, classes=5, n=600, in_dim=32, dropout=0.0, seed=0):
    edge = synth.powerlaw_graph(n, 5000, seed=3).to(dev)
    ei, adj = build_sparse_normalized_adjacency(edge, n)
    op = prepare_multihop_csr_operator(prepare_fixed_csr_operator(adj), dense_cols=2 * hidden)
    (rp, c), (r, cp), perm = to_graph_format(prepare_gat_edge_index(ei, n).flip(0), n)
    torch.manual_seed(seed)
    model = build_model(in_dim=in_dim, hidden_dim=hidden, out_dim=classes, num_layers=layers, dropout=dropout,
                        hop_scales=(1, 2, 3), gat_heads=2, gat_dropout=dropout).to(dev)
    model.prepare_fused_gat_graph(((rp, c), (r, cp), perm))
    g = torch.Generator(device=dev).manual_seed(7)
    x = torch.randn(n, in_dim, generator=g, device=dev)
    y = torch.randint(0, classes, (n,), generator=g, device=dev)
    labels = torch.where(torch.rand(n, generator=g, device=dev) < 0.5, y, torch.full_like(y, -1))
    return model, op, x, labels


def torch_loss(logits, labels, teacher=None, weight=0.5, temp=1.0, tail="drop"):
    z = logits.double()
    train = (labels >= 0).nonzero()[:, 0]
    loss = F.cross_entropy(z[train], labels[train])
    if teacher is None:
        return loss
    v, i = teacher[0].double(), teacher[1]
    logp = torch.log_softmax(z / temp, 1)
    if tail == "drop":
        q = torch.softmax(v / temp, 1)
        kl = (q * (q.log() - logp.gather(1, i))).sum(1)
    else:
        q = v.exp()
        kept = torch.zeros_like(logp, dtype=torch.bool).scatter_(1, i, True)
        rest = torch.logsumexp(logp.masked_fill(kept, -float("inf")), 1)
        r = 1 - q.sum(1)
        kl = (q * (v - logp.gather(1, i))).sum(1) + r * (r.log() - rest)
    return (1 - weight) * loss + weight * temp ** 2 * kl.mean()


@pytest.mark.parametrize("kind", ["labels", "drop", "bucket"])
def test_node_loss_and_gradients(cuda, kind):
    model, op, x, labels = setup(cuda)
    other, *_ = setup(cuda, seed=5)
    out = other.classify(x, op, top_k=2)
    teacher = None if kind == "labels" else (out.top_log_probs, out.top_index)
    temp = 2.0 if kind == "drop" else 1.0
    args = dict(teacher=teacher, distill_weight=0.3, temperature=temp, tail=kind) if teacher else {}
    loss = model.node_loss(x, op, labels, **args)
    grads = torch.autograd.grad(loss, list(model.parameters()))
    want = torch_loss(model(x, op), labels, teacher, 0.3, temp, kind)
    wgrads = torch.autograd.grad(want, list(model.parameters()))
    # a mean of some hundred values of order 1, each off by a few roundings of its log sum and of itself
    assert abs(float(loss.detach()) - float(want.detach())) <= 64 * U * (1 + abs(float(want.detach())))
    for (name, _), a, e in zip(model.named_parameters(), grads, wgrads):
        assert_parity(a, e, what=f"{kind} {name}")


def test_normalizer_is_that_of_the_whole_job(cuda):
    model, op, x, labels = setup(cuda)
    out = model.classify(x, op, top_k=3)
    teacher = (out.top_log_probs, out.top_index)
    whole = model.node_loss(x, op, labels, teacher, 0.5)
    count = int((labels >= 0).sum())
    again = model.node_loss(x, op, labels, teacher, 0.5, normalizer=(count, x.size(0)))
    half = model.node_loss(x, op, labels, teacher, 0.5, normalizer=(2 * count, 2 * x.size(0)))
    assert torch.equal(whole, again) and torch.equal(half * 2, again)
    nothing = model.node_loss(x, op, torch.full_like(labels, -1))
    assert float(nothing.detach()) == 0.0


def test_classify_is_the_models_softmax(cuda):
    model, op, x, labels = setup(cuda, dropout=0.5)
    model.train()
    out = model.classify(x, op, labels, 3)
    assert model.training and not out.log_prob.requires_grad
    model.eval()
    with torch.no_grad():
        logits = model(x, op)
    logp = torch.log_softmax(logits.double(), 1)
    order = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :3]
    assert torch.equal(out.top_index, order)
    assert float((out.top_log_probs - logp.gather(1, order)).abs().max()) <= 64 * U * 8


def test_wide_output_norm(cuda):
    """Five states of 512: wider than jk_layer_norm takes."""
    model, op, x, labels = setup(cuda, hidden=512, layers=4)
    torch_out = model(x, op)
    model.native_wide_norm = True
    native = model(x, op)
    assert_parity(native, torch_out, what="logits")
    ga = torch.autograd.grad(model.node_loss(x, op, labels), list(model.parameters()))
    model.native_wide_norm = False
    gb = torch.autograd.grad(model.node_loss(x, op, labels), list(model.parameters()))
    for (name, _), a, e in zip(model.named_parameters(), ga, gb):
        # two float32 norms of the same rows, each within 1e-5 of the exact one (assert_parity's bound)
        assert_parity(a, e, tol=2e-5, what=name)


def test_captured_distillation_step_replays_eager_ones(cuda):
    base, op, x, labels = setup(cuda)
    teacher_model, *_ = setup(cuda, seed=5)
    out = teacher_model.classify(x, op, top_k=3)
    teacher = (out.top_log_probs, out.top_index)

    def stepper(model):
        opt = torch.optim.Adam(model.parameters(), lr=0.01, capturable=True)

        def step():
            opt.zero_grad(set_to_none=True)
            loss = model.node_loss(x, op, labels, teacher, 0.5, tail="bucket")
            loss.backward()
            opt.step()
            return loss.detach()
        return step
    eager_model, graph_model = copy.deepcopy(base), copy.deepcopy(base)
    step = stepper(eager_model)
    eager = [float(step()) for _ in range(6)]
    graph = GraphedStep(stepper(graph_model), cuda, warmup=2)
    replayed = []
    for _ in range(4):
        replayed.append(float(graph()))
    assert replayed == eager[2:]
    for a, b in zip(graph_model.parameters(), eager_model.parameters()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d,c,k", [(300, 96, 47, 5), (64, 1000, 3001, 20)])
def test_the_operators_one_after_the_other(cuda, n, d, c, k, dtype):
    """norm -> classifier -> best classes of a teacher -> distillation and label loss of a student."""
    g = torch.Generator(device=cuda).manual_seed(n)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=cuda)
    x, labels = randn(n, d), torch.randint(-1, c, (n,), generator=g, device=cuda)
    leaves = [x, 1 + 0.1 * randn(d), 0.1 * randn(d), randn(c, d) / d ** 0.5, 0.1 * randn(c)]
    leaves = [t.to(dtype).requires_grad_() for t in leaves]
    teacher_logits = (randn(n, c) * 2).to(dtype)
    t = node_log_probs(teacher_logits, None, k)

    def chain(x, nw, nb, w, b):
        logits = F.linear(layer_norm(x, nw, nb), w, b)
        out = node_log_probs(logits, labels)
        kd = distill_top_logits(logits, t.top_log_probs, t.top_index, 1.0, "bucket")
        return logits, -out.log_prob.mean() - 0.01 * out.entropy.mean() + kd.mean()
    logits, loss = chain(*leaves)
    grads = torch.autograd.grad(loss, leaves)
    exact = [p.detach().double().requires_grad_() for p in leaves]
    # the chain's rounded logits enter the exact losses too, so that only the operators are compared
    z = F.linear(F.layer_norm(exact[0], (d,), exact[1], exact[2], 1e-5), exact[3], exact[4])
    z = z + (logits.detach().double() - z.detach())
    logp = torch.log_softmax(z, 1)
    at = labels.clamp(min=0)[:, None]
    ce = torch.where(labels >= 0, logp.gather(1, at)[:, 0], 0.0)
    entropy = -(logp.exp() * logp).sum(1)
    v = t.top_log_probs.double()
    kept = torch.zeros_like(logp, dtype=torch.bool).scatter_(1, t.top_index, True)
    r = 1 - v.exp().sum(1)
    kd = (v.exp() * (v - logp.gather(1, t.top_index))).sum(1) + \
        r * (r.log() - torch.logsumexp(logp.masked_fill(kept, -float("inf")), 1))
    want = -ce.mean() - 0.01 * entropy.mean() + kd.mean()
    assert abs(float(loss) - float(want)) <= 256 * U * (1 + abs(float(want)))
    wgrads = torch.autograd.grad(want, exact)
    # bf16: the logits' gradient, the classifier's products and the norm's output are each rounded to 2^-8 of
    # their size, and their errors add in the sums over rows: a few 2^-8 in all
    tol = 1e-5 if dtype == torch.float32 else 6 * 2.0 ** -8
    for a, e, what in zip(grads, wgrads, ("x", "norm weight", "norm bias", "weight", "bias")):
        assert_parity(a, e, tol=tol, what=what)
