"""distill_top_logits where teacher and student are far apart: kept classes that
the teacher all but rules out, classes that the student masks, both at once and
kept twice, over temperatures; against the definition in 64 bits."""
import pytest
import torch

from cign_b200.distill import distill_top_logits
from tests.class_rows import DTYPES
from tests.test_gpu_distill import INF, make, run_case
from tests.test_gpu_node_loss import setup

pytestmark = pytest.mark.gpu
LOW = torch.finfo(torch.float32).min
VALUES = (-12.0, -16.0, -90.0, -100.0, -200.0, -1e4, LOW)


def rule_out(x, v, i):
    """Row by row: the teacher's value of its best class (which the student prefers) becomes one of VALUES; so, and
    the student masks that class; that class is kept twice, once with its own value; both of its values are far and
    the student masks it."""
    for row in range(4 * len(VALUES)):
        value, kind = VALUES[row // 4], row % 4
        v[row, 0] = value
        if kind >= 2:
            i[row, 1] = i[row, 0]
        if kind == 3:
            v[row, 1] = value
        if kind in (1, 3):
            x[row, i[row, 0].long()] = -INF


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", [6, 60, 900, 20000])
@pytest.mark.parametrize("temp", [0.02, 1.0, 100.0])
def test_classes_that_the_teacher_rules_out(cuda, c, temp, dtype, tail):
    """The bounds of run_case hold as they are: a term q (e^-d - 1 + d) is p - q + q d, and p's rounding is that of
    its logarithm.  Where the student masks the class the loss is inf if q > 0 in 64 bits, and without q the
    class has no part in it."""
    for n in (28, 33, 41):
        run_case(cuda, n, c, 3, dtype, tail, temp, edit=rule_out)


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("c", [2, 600])
def test_two_classes_by_hand(cuda, c, tail):
    """Two classes at 0 (any others masked).  Drop: q = (1, 0), p = 1/2: loss log 2, gradient (-1/2, 1/2)."""
    for far in (-100.0, -104.0, -1e4, LOW):
        x = torch.full((1, c), -INF, device=cuda)
        x[0, :2] = 0.0
        x.requires_grad_()
        v, i = torch.tensor([[0.0, far]], device=cuda), torch.tensor([[0, 1]], device=cuda)
        loss = distill_top_logits(x, v, i, 1.0, tail)
        (grad,) = torch.autograd.grad(loss.sum(), x)
        assert abs(float(loss.detach()) - 0.6931471805599453) <= 4 * 2.0 ** -24
        assert (grad[0, :2].double() - torch.tensor([-0.5, 0.5], device=cuda)).abs().max() <= 4 * 2.0 ** -24
        assert not grad[0, 2:].any()


def test_both_mask_the_same_class(cuda):
    """A teacher's mask value beside a student's -inf: the class takes no part, as if it were absent."""
    for c in (7, 700):
        for tail in ("drop", "bucket"):
            x, v, i, _ = make(cuda, 2, c, 3, torch.float32, tail, 1.0)
            x[1], v[1], i[1] = x[0], v[0], i[0]
            x[:, i[0, 2]] = -INF
            v[0, 2], v[1, 2] = -1e4, -INF
            if tail == "bucket":
                v[:, :2] = torch.log_softmax(v[:, :2], 1)  # no rest, whose classes differ
                v[:, :2] += 1e-6
            x.requires_grad_()
            loss = distill_top_logits(x, v, i, 1.0, tail)
            (grad,) = torch.autograd.grad(loss.sum(), x)
            assert torch.isfinite(loss).all() and torch.equal(loss[0], loss[1]) and torch.equal(grad[0], grad[1])


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("c", [6, 60, 900, 20000])
def test_a_value_that_is_no_number_makes_its_row_so(cuda, c, tail):
    x, v, i, _ = make(cuda, 9, c, 3, torch.float32, tail, 1.0)
    v[1, 0] = v[2, 2] = float("nan")
    v[3] = float("nan")
    v[4, 1], i[4, 1] = float("nan"), -1  # absent
    x.requires_grad_()
    loss = distill_top_logits(x, v, i, 1.0, tail)
    (grad,) = torch.autograd.grad(loss, x, torch.ones(9, device=cuda))
    assert torch.isnan(loss).tolist() == [r in (1, 2, 3) for r in range(9)]
    assert torch.isnan(grad).any(1).tolist() == [r in (1, 2, 3) for r in range(9)]


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", [6, 60, 900])
@pytest.mark.parametrize("temp", [0.005, 0.02, 0.05])
def test_low_temperatures(cuda, c, temp, dtype, tail):
    """Many rows in which a gap of a few between the teacher's logits that the student does not share is a
    probability of less than e^-88."""
    for n in (100, 101, 307):
        run_case(cuda, n, c, 4, dtype, tail, temp)


def test_one_such_node_does_not_spoil_a_training_step(cuda):
    model, op, x, labels = setup(cuda)
    other, *_ = setup(cuda, seed=5)
    out = other.classify(x, op, top_k=3)
    values = out.top_log_probs.clone()
    values[17, 0] = -1e4
    values[18, 1] = -100.0
    for tail in ("drop", "bucket"):
        loss = model.node_loss(x, op, labels, (values, out.top_index), 0.5, tail=tail)
        grads = torch.autograd.grad(loss, list(model.parameters()))
        assert torch.isfinite(loss) and all(torch.isfinite(g).all() for g in grads)
