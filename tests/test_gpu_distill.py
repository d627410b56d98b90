"""distill_top_logits against the divergence's definition in 64 bits: loss and
gradient for both tails, types, layouts, absent and repeated entries, near and
far teachers, masked students, row counts, streams and captured graphs."""
import pytest
import torch

from cign_b200.distill import distill_top_logits
from cign_b200.graph_step import GraphedStep
from cign_b200.node_log_probs import node_log_probs
from tests.class_rows import DTYPES, U, check, layout, sum_ulps

pytestmark = pytest.mark.gpu
INF = float("inf")


def index_layout(i, dtype, kind):
    if kind != "padded":
        return i.to(dtype)
    buf = torch.full((i.size(0), i.size(1) + 3), -1, dtype=dtype, device=i.device)
    buf[:, :i.size(1)] = i
    return buf[:, :i.size(1)]


def make(dev, n, c, k, dtype, tail, temp, kind="plain", noise=1.0, vdtype=torch.float32, idtype=torch.int64):
    g = torch.Generator(device=dev).manual_seed(n * 31 + c + k)
    x = torch.randn(n, c, generator=g, device=dev) * 2
    x[torch.arange(n, device=dev), torch.randint(0, c, (n,), generator=g, device=dev)] += 6.0
    t = x + noise * torch.randn(n, c, generator=g, device=dev)
    if tail == "bucket":
        t = torch.log_softmax(t / temp, 1)
    v, i = t.topk(k, dim=1)
    return layout(x, dtype, kind), layout(v, vdtype, kind), index_layout(i, idtype, kind), g


def reference(x, v, i, temp, tail, g):
    """loss, grad and what their errors are measured by; rows must have an entry."""
    c = x.size(1)
    x, v, i, g = x.detach().double(), v.double(), i.long(), g.double()
    z = x / temp
    logp = torch.log_softmax(z, 1)
    p = logp.exp()
    here = (i >= 0) & (v > -INF)
    at = i.clamp(min=0)
    if tail == "drop":
        v = torch.log_softmax(torch.where(here, v, -INF) / temp, 1)
    q = torch.where(here, v.exp(), 0.0)
    kept = torch.zeros_like(p).scatter_add_(1, at, here.double()) > 0
    target = torch.zeros_like(p).scatter_add_(1, at, q)
    delta = torch.where(here, v - logp.gather(1, at), 0.0)
    loss = torch.where(q > 0, q * delta, 0.0).sum(1)
    p_rest = torch.where(kept, 0.0, p).sum(1)
    mass, r = q.sum(1), torch.zeros_like(loss)
    if tail == "bucket":
        r = torch.where(kept.all(1), 0.0, (1 - mass).clamp(min=0.0))
        # by logarithms: p_rest may be far below what its exponentials can hold
        log_rest = torch.logsumexp(logp.masked_fill(kept, -INF), 1)
        loss = loss + torch.where(r > 0, r * (r.log() - log_rest), 0.0)
        spread = torch.where(kept | (logp == -INF), 0.0, r[:, None] * (logp - log_rest[:, None]).exp())
    else:
        spread = torch.zeros_like(p)
    W = mass + r
    grad = W[:, None] * p - target - spread
    grad = grad * temp * g[:, None]
    # k roundings on the way of each probability (and below 2^-126, the smallest normal number, an exponential is
    # 0, so a gradient is off by up to that); those of the log sum cancel in the loss to first order, what is left
    # is weighted with |p - q|, which is at most sqrt(2 KL) in all (Pinsker)
    d = torch.where(torch.isfinite(z), z.amax(1, keepdim=True) - z, 0.0)
    ku = 2 * (sum_ulps(c) + sum_ulps(i.size(1)) + 16) * U
    dmax = (p * (1 + d)).sum(1) + 1
    kl = loss + (1 - W)  # of the two full distributions, never negative
    away = (2 * kl.clamp(min=0)).sqrt() + (W - 1).abs()
    tloss = temp ** 2 * (ku * (loss.abs() + kl.abs()) + ku * dmax * (away + away ** 2) + (ku * dmax) ** 2 + U * (1 - W).abs())
    # entries of one class are not a distribution over classes: besides one term q (d - 1 + e^-d) of a class they
    # leave terms q (d - 1) of either sign, whose roundings count with their magnitudes
    twice = (kept.sum(1) < here.sum(1))
    tloss = tloss + torch.where(twice, temp ** 2 * ku * torch.where(q > 0, q * (1 + delta.abs()), 0.0).sum(1), 0.0)
    tgrad = temp * g.abs()[:, None] * (2.0 ** -125 + ku * (dmax[:, None] + d) * (p + spread)
                                       + ku * (target + (W[:, None] * p - target).abs()))
    return temp ** 2 * loss, grad, tloss, tgrad


def run_case(dev, n, c, k, dtype, tail, temp=2.0, edit=None, **kw):
    x, v, i, gen = make(dev, n, c, k, dtype, tail, temp, **kw)
    if edit is not None:
        edit(x, v, i)
    x.requires_grad_()
    g = 0.5 + torch.rand(n, generator=gen, device=dev)
    want, wgrad, tl, tg = reference(x, v, i, temp, tail, g)
    loss = distill_top_logits(x, v, i, temp, tail)
    what = f"n={n} c={c} k={k} {dtype} {tail} T={temp} {kw}"
    assert loss.dtype == torch.float32 and loss.shape == (n,)
    check(loss, want, tl, f"loss {what}")
    (grad,) = torch.autograd.grad(loss, x, g)
    assert grad.dtype == dtype
    check(grad, wgrad, tg, f"grad {what}")


SIZES = [(1, 1, 1), (3, 2, 1), (24, 5, 2), (30, 5, 5), (100, 7, 3), (33, 16, 16), (65, 31, 4), (40, 33, 20), (500, 47, 5),
         (77, 64, 64), (20, 100, 33), (9, 129, 100), (7, 257, 200), (11, 256, 256), (5, 512, 20), (6, 513, 64), (4, 1000, 8),
         (3, 1025, 256), (200, 1500, 20), (3, 4099, 65), (2, 10007, 20), (1, 50001, 100), (2, 131072, 64)]


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,c,k", SIZES)
def test_loss_and_gradient(cuda, n, c, k, dtype, tail):
    run_case(cuda, n, c, k, dtype, tail)


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("temp", [0.5, 1.0, 3.0])
@pytest.mark.parametrize("n,c,k", [(300, 6, 3), (40, 90, 10), (9, 3000, 20)])
def test_temperatures_and_near_teachers(cuda, n, c, k, temp, tail):
    run_case(cuda, n, c, k, torch.float32, tail, temp)
    run_case(cuda, n, c, k, torch.float32, tail, temp, noise=0.01)


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("kind", ["padded", "shifted"])
@pytest.mark.parametrize("n,c,k", [(50, 5, 2), (33, 47, 5), (9, 300, 20), (3, 30011, 64)])
def test_layouts_and_types(cuda, n, c, k, kind, tail):
    for dtype, vdtype, idtype in ((torch.float32, torch.float32, torch.int32), (torch.bfloat16, torch.float16, torch.int64),
                                  (torch.float16, torch.bfloat16, torch.int32)):
        run_case(cuda, n, c, k, dtype, tail, kind=kind, vdtype=vdtype, idtype=idtype)


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("c,k", [(40, 6), (700, 20), (20000, 64)])
def test_absent_and_repeated_entries(cuda, c, k, tail):
    def absent(x, v, i):
        i[0, 1:] = -1
        v[1, 3:] = -INF
        i[2, ::2] = -100
        v[2, 1] = -INF

    def repeated(x, v, i):
        i[0, 1] = i[0, 0]
        i[1, :] = i[1, 0]
        i[2, 5] = i[2, 2]
        i[2, 4] = i[2, 2]
        v[3, 1] = -INF
        i[3, 1] = i[3, 0]
    for dtype in DTYPES:
        run_case(cuda, 5, c, k, dtype, tail, edit=absent)
        run_case(cuda, 5, c, k, dtype, tail, edit=repeated)


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("c", [5, 60, 900, 20000])
def test_rows_without_entries_and_wrong_classes(cuda, c, tail):
    k = 4
    x, v, i, _ = make(cuda, 7, c, k, torch.float32, tail, 1.0)
    i[1] = -1
    v[2] = -INF
    i[3, 2] = c
    i[4, 0] = 2 ** 33
    x[1, 0] = float("nan")   # no teacher, so what the student holds is not looked at
    x[5, c - 1] = float("nan")
    x[6, 0] = INF
    x.requires_grad_()
    loss = distill_top_logits(x, v, i, 1.0, tail)
    assert loss[1] == 0 and loss[2] == 0
    assert torch.isnan(loss).tolist() == [False, False, False, True, True, True, True]
    (grad,) = torch.autograd.grad(loss, x, torch.ones(7, device=cuda))
    assert not grad[1].any() and not grad[2].any() and torch.isfinite(grad[0]).all()
    assert torch.isnan(grad[3:]).all()
    # rows that no gradient reaches
    (grad,) = torch.autograd.grad(distill_top_logits(x, v, i, 1.0, tail), x, torch.zeros(7, device=cuda))
    assert not grad.any()


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("c", [5, 60, 900, 20000])
def test_masked_students(cuda, c, tail):
    k = 3
    x, v, i, _ = make(cuda, 6, c, k, torch.float32, tail, 1.0)
    low = torch.finfo(torch.float32).min
    kept = torch.zeros(6, c, dtype=torch.bool, device=cuda).scatter_(1, i, True)
    x[1] = -INF                                    # nothing left
    x[2] = torch.where(kept[2], x[2], -INF)        # only kept classes left
    x[3, i[3, 1]] = -INF                           # a kept class is masked
    x[4] = low                                     # masked by the lowest value: uniform
    x[5] = torch.where(kept[5], x[5], low)
    x.requires_grad_()
    loss = distill_top_logits(x, v, i, 1.0, tail)
    (grad,) = torch.autograd.grad(loss, x, torch.ones(6, device=cuda))
    want, wgrad, tl, tg = reference(x[[0, 3, 4]], v[[0, 3, 4]], i[[0, 3, 4]], 1.0, tail, torch.ones(3, device=cuda))
    assert loss[1] == INF and loss[3] == INF and not grad[1].any()
    check(loss[[0, 4]], want[[0, 2]], tl[[0, 2]], "loss")
    check(grad[[0, 3, 4]], wgrad, torch.where(torch.isfinite(tg), tg, 64 * U), "grad")
    for row in (2, 5):
        # the others have probability 0: with a rest to place the divergence is infinite (row 2), or, as the
        # lowest value is finite, r times its distance
        if tail == "bucket" and row == 2:
            assert loss[row] == INF
        else:
            e, eg, te, tge = reference(x[row:row + 1, :], v[row:row + 1], i[row:row + 1], 1.0, tail, torch.ones(1, device=cuda))
            check(loss[row:row + 1], e, te, "loss")
            check(grad[row:row + 1], eg, tge, "grad")
    assert not torch.isnan(grad).any()


@pytest.mark.parametrize("n", [149, 1000, 6000])
@pytest.mark.parametrize("c", [40, 700, 3001])
def test_row_counts(cuda, n, c):
    run_case(cuda, n, c, 8, torch.float32, "drop")
    run_case(cuda, n, c, 8, torch.bfloat16, "bucket")


def test_equal_distributions_have_no_divergence(cuda):
    """The student is the teacher: loss and gradient vanish to the second order of the roundings."""
    for c, k in ((5, 2), (60, 10), (900, 64), (30000, 64)):
        x = torch.randn(4, c, device=cuda) * 3
        out = node_log_probs(x, None, k)
        x.requires_grad_()
        loss = distill_top_logits(x, out.top_log_probs, out.top_index, 1.0, "bucket")
        assert bool((loss.abs() <= 1e-10).all()) and bool((loss >= 0).all())


def test_all_classes_kept_is_the_whole_divergence(cuda):
    n, c = 50, 12
    x, v, i, g = make(cuda, n, c, c, torch.float32, "bucket", 1.0, noise=0.3)
    x.requires_grad_()
    t = torch.empty(n, c, device=cuda, dtype=torch.float64).scatter_(1, i, v.double())
    want = (t.exp() * (t - torch.log_softmax(x.detach().double(), 1))).sum(1)
    room = 512 * U * ((2 * want.abs()).sqrt() + want.abs()) + 64 * U * (1 - t.exp().sum(1)).abs() + (256 * U) ** 2
    check(distill_top_logits(x, v, i, 1.0, "bucket"), want, room, "bucket")
    check(distill_top_logits(x, v, i, 1.0, "drop"), want, room + 2 * (1 - t.exp().sum(1)).abs(), "drop")


def test_gradient_against_differences(cuda):
    for tail in ("drop", "bucket"):
        x, v, i, g = make(cuda, 8, 30, 5, torch.float32, tail, 2.0)
        w = torch.rand(8, generator=g, device=cuda)
        x.requires_grad_()
        (grad,) = torch.autograd.grad(distill_top_logits(x, v, i, 2.0, tail), x, w)
        h = 2.0 ** -5
        d = torch.randn(8, 30, generator=g, device=cuda)
        d = d / d.norm()

        def loss(t):
            return float((distill_top_logits(t, v, i, 2.0, tail).double() * w).sum())
        diff = (loss(x.detach() + h * d) - loss(x.detach() - h * d)) / (2 * h)
        top = float(distill_top_logits(x.detach(), v, i, 2.0, tail).max())
        assert abs(diff - float((grad.double() * d.double()).sum())) <= float(w.sum()) * (8 * h * h / 6 + 64 * U * (1 + top) / h)


def test_broadcast_gradient_and_constant_teacher(cuda):
    x, v, i, _ = make(cuda, 90, 200, 6, torch.float32, "drop", 1.0)
    x.requires_grad_()
    loss = distill_top_logits(x, v, i)
    (a,) = torch.autograd.grad(loss.sum(), x, retain_graph=True)
    (b,) = torch.autograd.grad(loss, x, torch.ones(90, device=cuda))
    assert torch.equal(a, b)
    one = distill_top_logits(x, v[:1].expand(90, 6), i[:1].expand(90, 6))
    assert torch.equal(one, distill_top_logits(x, v[:1].repeat(90, 1), i[:1].repeat(90, 1)))
    with pytest.raises(ValueError):
        distill_top_logits(x, v.requires_grad_(), i)


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", [6, 60, 900, 20000])
@pytest.mark.parametrize("temp", [0.02, 500.0, 20000.0])
def test_far_temperatures_and_masks(cuda, c, temp, dtype, tail):
    """Masked classes have no probability at any temperature; far logits come near at a high one."""
    def edit(x, v, i):
        kept = torch.zeros_like(x, dtype=torch.bool).scatter_(1, i.long(), True)
        x[0] = torch.where(kept[0], x[0], torch.full_like(x[0], -INF))  # all but the kept ones
        x[1, :c // 2] = torch.where(kept[1, :c // 2], x[1, :c // 2], torch.full_like(x[1, :c // 2], -INF))
        x[2] *= 300.0
        if tail == "bucket":
            v[0] += 0.2 / 3  # nothing to place on masked classes
            v[0] -= torch.logsumexp(v[0], 0)
    if tail == "bucket":
        # row 0 has no rest: r is 1 - sum q, a rounding; only the loss of a rest that exists is compared
        x, v, i, gen = make(cuda, 4, c, 3, dtype, tail, temp)
        edit(x, v, i)
        want, wgrad, tl, tg = reference(x[1:], v[1:], i[1:], temp, tail, torch.ones(3, device=cuda))
        x.requires_grad_()
        loss = distill_top_logits(x, v, i, temp, tail)
        (grad,) = torch.autograd.grad(loss[1:].sum(), x)
        check(loss[1:], want, tl, "loss")
        check(grad[1:], wgrad, tg, "grad")
        assert not grad[0].any()
    else:
        run_case(cuda, 4, c, 3, dtype, tail, temp, edit=edit)


def test_empty(cuda):
    x = torch.zeros(0, 9, device=cuda, requires_grad=True)
    loss = distill_top_logits(x, torch.zeros(0, 2, device=cuda), torch.zeros(0, 2, dtype=torch.int32, device=cuda))
    (grad,) = torch.autograd.grad(loss.sum(), x)
    assert grad.shape == (0, 9) and loss.shape == (0,)


def test_repeats_bit_for_bit_on_streams_and_in_graphs(cuda):
    x, v, i, _ = make(cuda, 400, 3000, 20, torch.bfloat16, "bucket", 1.0)
    i[5, 3] = i[5, 0]
    x.requires_grad_()
    out = {}

    def step():
        loss = distill_top_logits(x, v, i, 1.0, "bucket")
        (out["g"],) = torch.autograd.grad(loss.sum(), x)
        out["l"] = loss.detach()
        return out["l"]
    step()
    first = [out["l"].clone(), out["g"].clone()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out["l"], first[0]) and torch.equal(out["g"], first[1])
    graph = GraphedStep(step, cuda, warmup=2)
    captured = [out["l"], out["g"]]
    for _ in range(2):
        graph()
        torch.cuda.synchronize()
        assert torch.equal(captured[0], first[0]) and torch.equal(captured[1], first[1])


def test_second_derivative_is_refused(cuda):
    x, v, i, _ = make(cuda, 4, 8, 2, torch.float32, "drop", 1.0)
    x.requires_grad_()
    (g,) = torch.autograd.grad(distill_top_logits(x, v, i).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_refusals(cuda):
    x, v, i, _ = make(cuda, 4, 300, 6, torch.float32, "drop", 1.0)
    for args, error in (((x.double(), v, i), TypeError), ((x.cpu(), v, i), TypeError), ((x, v.double(), i), TypeError),
                        ((x, v, i.float()), TypeError), ((x, v.cpu(), i), TypeError), ((x, v, i[:, :5]), ValueError),
                        ((x, v[:3], i[:3]), ValueError), ((x, v[:, :0], i[:, :0]), ValueError), ((x[0], v, i), ValueError),
                        ((x, v, i, 0.0), ValueError), ((x, v, i, float("inf")), ValueError), ((x, v, i, float("nan")), ValueError),
                        ((x, v, i, 1e-4), ValueError), ((x, v, i, 2e6), ValueError), ((x, v, i, 1.0, "rest"), ValueError),
                        ((x, v[:, :1].expand(4, 257), i[:, :1].expand(4, 257)), ValueError)):
        with pytest.raises(error):
            distill_top_logits(*args)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", [6, 60, 900, 30000])
def test_far_rest_keeps_its_share(cuda, c, dtype):
    """The student's other classes are e^-95 and e^-190 below its kept ones, less than float32 can hold: the rest's
    part of the loss and its gradient are those of the logarithms."""
    k = 3
    x, v, i, gen = make(cuda, 4, c, k, torch.float32, "bucket", 1.0)
    kept = torch.zeros(4, c, dtype=torch.bool, device=cuda).scatter_(1, i, True)
    gap = torch.tensor([[30.0], [95.0], [190.0], [60.0]], device=cuda)
    x = torch.where(kept, x, x - gap).to(dtype).requires_grad_()
    v = v - 0.5
    g = 0.5 + torch.rand(4, generator=gen, device=cuda)
    want, wgrad, tl, tg = reference(x, v, i, 1.0, "bucket", g)
    # the gradient of the others is r times their distribution among themselves, known to the roundings of the
    # exponents, which are relative to the gap
    rest = torch.where(kept, 0.0, torch.softmax(x.detach().double().masked_fill(kept, -INF), 1))
    tg = torch.where(kept, tg, 512 * U * (1 + gap.double() / 8) * rest * g.double()[:, None])
    loss = distill_top_logits(x, v, i, 1.0, "bucket")
    check(loss, want, 512 * U * want.abs(), "loss")
    (grad,) = torch.autograd.grad(loss, x, g)
    check(grad, wgrad, tg, "grad")
