"""node_log_probs against log softmax in 64 bits: values, best classes in
order, gradients, masked classes and rows, missing and wrong labels, layouts,
row counts from one to many, streams and captured graphs."""
import pytest
import torch

from cign_b200.graph_step import GraphedStep
from cign_b200.node_log_probs import NodeLogProbs, node_log_probs
from tests.class_rows import DTYPES, U, check, layout, sum_ulps

pytestmark = pytest.mark.gpu
INF = float("inf")


def make(dev, n, c, dtype, kind="plain", masked=0.0, seed=0, spread=2.0):
    g = torch.Generator(device=dev).manual_seed(seed + n * 31 + c)
    x = torch.randn(n, c, generator=g, device=dev) * spread
    x[torch.arange(n, device=dev), torch.randint(0, c, (n,), generator=g, device=dev)] += 8.0
    labels = torch.randint(0, c, (n,), generator=g, device=dev)
    if masked:
        hide = torch.rand(n, c, generator=g, device=dev) < masked
        hide[torch.arange(n, device=dev), labels] = False
        x = x.masked_fill(hide, -INF)
    labels = torch.where(torch.rand(n, generator=g, device=dev) < 0.2, torch.full_like(labels, -100), labels)
    return layout(x, dtype, kind), labels, g


def reference(x, labels):
    x = x.detach().double()
    logp = torch.log_softmax(x, 1)
    p = logp.exp()
    plogp = torch.where(p > 0, p * logp, 0.0)
    at = labels.clamp(min=0)
    lp = torch.where(labels >= 0, logp.gather(1, at[:, None])[:, 0], 0.0)
    return logp, p, lp, -plogp.sum(1)


def far(x):
    """How far below the row's maximum the finite logits are: the relative error of e^(x - m)
    is (2 + |x - m|) float32 roundings, twice that where a hardware exponential is used."""
    d = (x.detach().double().amax(1, keepdim=True) - x.detach().double())
    return torch.where(torch.isfinite(d), d, 0.0)


def run_case(dev, n, c, dtype, kind="plain", masked=0.0, top_k=0, spread=2.0):
    x, labels, g = make(dev, n, c, dtype, kind, masked, spread=spread)
    x.requires_grad_()
    logp, p, lp, H = reference(x, labels)
    out = node_log_probs(x, labels, top_k)
    k = 2 * (sum_ulps(c) + 16) * U
    what = f"n={n} c={c} {dtype} {kind} k={top_k}"
    d = far(x)
    # log1p(s): the relative errors of the terms of s, weighted with their share of 1 + s; the maximum's own 1 is exact
    others = p.scatter(1, p.argmax(1, keepdim=True), 0.0)
    sum_err = k * (others * (1 + d)).sum(1)
    check(out.log_prob, lp, torch.where(labels >= 0, sum_err + 4 * U * d.gather(1, labels.clamp(min=0)[:, None])[:, 0] + 4 * U * lp.abs(), 0.0), f"log_prob {what}")
    check(out.entropy, H, k * (H + (p * d * (1 + d)).sum(1)), f"entropy {what}")
    if top_k:
        order = torch.sort(x.detach().float(), dim=1, descending=True, stable=True)[1][:, :top_k]
        assert torch.equal(out.top_index, order), f"top {what}"
        want = logp.gather(1, order)
        check(out.top_log_probs, want, sum_err[:, None] + 4 * U * (d.gather(1, order) + torch.where(torch.isfinite(want), want.abs(), 0.0)), f"top {what}")
    # gradients of all outputs
    gl = torch.randn(n, generator=g, device=dev)
    gh = 0.3 * torch.randn(n, generator=g, device=dev)
    outs, ups = [out.log_prob, out.entropy], [gl, gh]
    G = torch.where(labels >= 0, gl.double(), 0.0)
    a = torch.zeros_like(p).scatter_add_(1, labels.clamp(min=0)[:, None], G[:, None])
    if top_k:
        gt = torch.randn(n, top_k, generator=g, device=dev)
        gt = torch.where(torch.isfinite(out.top_log_probs), gt, torch.zeros_like(gt))
        outs.append(out.top_log_probs)
        ups.append(gt)
        a = a.scatter_add(1, out.top_index, gt.double())
        G = G + gt.double().sum(1)
    (grad,) = torch.autograd.grad(outs, x, ups)
    assert grad.dtype == dtype
    lpz = torch.where(p > 0, logp, 0.0)
    want = a - p * G[:, None] - gh.double()[:, None] * p * (lpz + H[:, None])
    absG = G.abs() if not top_k else G.abs() + gt.double().abs().sum(1)
    room = p * (k + 4 * U * d + 4 * U * lpz.abs()) * (absG[:, None] + gh.double().abs()[:, None] * (1 + lpz.abs() + H[:, None])) + 4 * U * (a.abs() + torch.where(a != 0, absG[:, None] * (1 - p), 0.0))
    if top_k:
        room = room + torch.where(a != 0, (top_k + 4) * U * absG[:, None], 0.0)
    check(grad, want, room, f"grad {what}")


SIZES = [(1, 1), (3, 2), (24, 5), (100, 7), (65, 16), (129, 31), (40, 32), (41, 33), (1000, 47), (77, 64),
         (50, 100), (33, 128), (9, 129), (30, 256), (7, 257), (20, 500), (5, 512), (6, 513), (4, 1000),
         (3, 1024), (5, 1025), (200, 1500), (3, 4099), (2, 10007), (1, 50001), (3, 131072)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,c", SIZES)
def test_values_and_gradients(cuda, n, c, dtype):
    run_case(cuda, n, c, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,c,k", [(3, 1, 1), (50, 5, 3), (50, 5, 5), (33, 47, 20), (20, 64, 64), (9, 100, 33),
                                   (7, 300, 64), (5, 1000, 1), (5, 1500, 32), (4, 5000, 31), (3, 10007, 64),
                                   (300, 2049, 20), (1, 70001, 8), (2, 131071, 64)])
def test_best_classes(cuda, n, c, k, dtype):
    run_case(cuda, n, c, dtype, top_k=k)
    run_case(cuda, n, c, dtype, kind="padded", top_k=k, masked=0.3 if c > 2 * k else 0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["padded", "shifted"])
@pytest.mark.parametrize("n,c", [(50, 5), (33, 47), (9, 300), (5, 2000), (3, 30011)])
def test_layouts_and_masks(cuda, n, c, kind, dtype):
    run_case(cuda, n, c, dtype, kind, masked=0.5)


@pytest.mark.parametrize("n", [149, 296, 1000, 5000])
@pytest.mark.parametrize("c", [40, 700, 3001])
def test_row_counts(cuda, n, c):
    run_case(cuda, n, c, torch.float32, top_k=4)
    run_case(cuda, n, c, torch.bfloat16)


@pytest.mark.parametrize("c", [6, 200, 3000, 40000])
def test_equal_logits_go_to_the_lower_class(cuda, c):
    k = min(c, 64)
    for value in (0.0, -INF, -3.0e38, 5.0):
        x = torch.full((3, c), value, device=cuda)
        x[1, ::2] = -0.0 if value == 0.0 else value
        out = node_log_probs(x, None, k)
        assert torch.equal(out.top_index, torch.arange(k, device=cuda).expand(3, k))
    g = torch.Generator(device=cuda).manual_seed(c)
    x = torch.randint(-3, 3, (5, c), generator=g, device=cuda).float()  # few values, many ties
    x[2] = torch.arange(c, device=cuda) * 0.01   # every next class is better
    x[3] = -x[2]
    order = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :k]
    assert torch.equal(node_log_probs(x, None, k).top_index, order)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [4, 5, 6, 10, 11, 17, 32, 33, 64])
@pytest.mark.parametrize("c", [65, 97, 128, 129, 193, 256, 257, 385, 512])
def test_best_classes_of_narrow_rows(cuda, c, k, dtype):
    """Rows of different kinds side by side in a warp, the last warp not full: plain ones, few values with ties at
    the border, masked, all masked, NaN, +inf, far magnitudes, all equal, values next to each other."""
    g = torch.Generator(device=cuda).manual_seed(c * 100 + k)
    n = 41
    x = torch.randn(n, c, generator=g, device=cuda)
    x[1::9] = torch.randint(-2, 3, (x[1::9].size(0), c), generator=g, device=cuda).float()
    x[2::9] = x[2::9].masked_fill(torch.rand(x[2::9].shape, generator=g, device=cuda) < 0.97, -INF)
    x[3::9] = -INF
    x[4::9, 7::30] = float("nan")
    x[5::9, 11] = INF
    x[6::9] *= 60000.0
    x[6::9] = x[6::9].clamp(-65504, 65504)
    x[7::9] = 0.25
    x[8::9] = 1.0 + torch.arange(c, device=cuda).flip(0) * torch.finfo(dtype).eps
    x = x.to(dtype)
    out = node_log_probs(x, None, k)
    order = torch.sort(x.float(), dim=1, descending=True, stable=True)[1][:, :k]
    assert torch.equal(out.top_index, order)
    z = x.double()
    best = z.gather(1, order)
    lp = torch.where(torch.isinf(z).all(1, keepdim=True) & (z < 0).all(1, keepdim=True), -INF,
                     best - torch.logsumexp(z, 1, keepdim=True))
    lp = torch.where((torch.isnan(z) | (z == INF)).any(1, keepdim=True), float("nan"), lp)
    # the sum's roundings, and those of x - m and of the difference to the logarithm
    check(out.top_log_probs, lp, (c / 256 + 24) * U * (1 + torch.where(torch.isfinite(lp), lp.abs(), 0.0)), "top")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,c,k", [(4, 30, 10), (4, 300, 40), (300, 5000, 64), (2, 70001, 20), (4000, 1500, 50)])
def test_fewer_classes_left_than_asked_for(cuda, n, c, k, dtype):
    """All but three classes are masked: the best are these, then masked ones by their index."""
    g = torch.Generator(device=cuda).manual_seed(c)
    x = torch.full((n, c), -INF, device=cuda, dtype=dtype)
    at = torch.rand(n, c, generator=g, device=cuda).topk(3, 1)[1]
    x.scatter_(1, at, torch.randn(n, 3, generator=g, device=cuda).to(dtype))
    out = node_log_probs(x, None, k)
    order = torch.sort(x.float(), dim=1, descending=True, stable=True)[1][:, :k]
    assert torch.equal(out.top_index, order)
    logp = torch.log_softmax(x.double(), 1).gather(1, order)
    check(out.top_log_probs, logp, 64 * U * (1 + torch.where(torch.isfinite(logp), logp.abs(), 0.0)), "top")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", [1, 5, 90, 600, 20000])
def test_masked_rows_and_lowest_values(cuda, c, dtype):
    low = torch.finfo(dtype).min
    x = torch.zeros(5, c, dtype=dtype, device=cuda)
    x[0] = -INF
    x[1] = -INF
    x[2] = low          # masked by the type's lowest value: a uniform row
    x[3] = low
    x[3, c - 1] = torch.finfo(dtype).max
    labels = torch.tensor([c - 1, -1, 0, c - 1, 0], device=cuda)
    x.requires_grad_()
    out = node_log_probs(x, labels, 1)
    logc = torch.tensor(float(c), dtype=torch.float64).log().item()
    want = torch.tensor([-INF, 0.0, -logc, 0.0, -logc], device=cuda)
    check(out.log_prob, want, sum_ulps(c) * U * (1 + logc), "log_prob")
    check(out.entropy, torch.tensor([0.0, 0.0, logc, 0.0, logc], device=cuda), sum_ulps(c) * U * (1 + logc), "entropy")
    assert out.top_index[:, 0].tolist() == [0, 0, 0, c - 1, 0]
    assert out.top_log_probs[0].item() == -INF and out.top_log_probs[3].item() == 0.0
    (grad,) = torch.autograd.grad((out.log_prob, out.entropy), x, (torch.ones(5, device=cuda), torch.ones(5, device=cuda)))
    assert not grad[0].any() and not grad[1].any() and not grad[3].any()
    assert torch.isfinite(grad).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", [6, 90, 900, 20000])
def test_far_logits(cuda, c, dtype):
    """Rows far from 0: all equal, two values a step apart, a mask of -1e4 and a spread of thousands."""
    big = 3.0e4 if dtype == torch.float16 else 1.0e20
    x = torch.full((6, c), -big, device=cuda, dtype=dtype)
    x[1] = big
    x[2] = torch.where(torch.arange(c, device=cuda) % 3 == 0, 2048.0, 2040.0)
    x[3] = torch.where(torch.arange(c, device=cuda) % 2 == 0, -1e4, 1.0)
    x[4] = torch.linspace(-3e3, 3e3, c, device=cuda)
    x[5] = torch.where(torch.arange(c, device=cuda) % 3 == 0, 30000.0, 29968.0)
    labels = torch.tensor([0, 1, 3, 1, c - 1, 0], device=cuda)
    x = x.to(dtype).requires_grad_()
    logp, p, lp, H = reference(x, labels)
    out = node_log_probs(x, labels, 2)
    k = 2 * (sum_ulps(c) + 16) * U
    check(out.log_prob, lp, k * (1 + lp.abs()), "log_prob")
    check(out.entropy, H, k * (1 + H), "entropy")
    g = torch.ones(6, device=cuda)
    (grad,) = torch.autograd.grad((out.log_prob, out.entropy), x, (g, g))
    plogp = torch.where(p > 0, p * (logp + H[:, None]), 0.0)
    want = torch.zeros_like(p).scatter_(1, labels[:, None], 1.0) - p - plogp
    # 16 bits: the exponent's shift is rounded to 2^-11 at most, below half a step of the gradient
    room = (k + (2.0 ** -11 if dtype != torch.float32 else 0.0)) * (p * (1 + torch.where(p > 0, (logp + H[:, None]).abs(), 0.0)))
    check(grad, want, room + 8 * U * (1 - p).clamp(min=0) * (want > 0), "grad")


@pytest.mark.parametrize("c", [4, 90, 3000, 20001])
def test_nan_infinity_and_wrong_labels(cuda, c):
    x = torch.randn(6, c, device=cuda)
    x[1, c - 1] = float("nan")
    x[2, c // 2] = INF
    labels = torch.tensor([0, 0, 0, c, 2 ** 40, -7], device=cuda)
    x.requires_grad_()
    out = node_log_probs(x, labels, 2)
    assert torch.isnan(out.log_prob).tolist() == [False, True, True, True, True, False]
    assert torch.isnan(out.entropy).tolist() == [False, True, True, False, False, False]
    assert out.top_index[1, 0].item() == c - 1 and out.top_index[2, 0].item() == c // 2
    (grad,) = torch.autograd.grad(out.log_prob, x, torch.ones(6, device=cuda))
    assert torch.isnan(grad).all(1).tolist() == [False, True, True, True, True, False]
    assert torch.isfinite(grad[0]).all() and not grad[5].any()
    # a row that no gradient reaches is left alone whatever it holds
    w = torch.tensor([1.0, 0, 0, 0, 0, 0], device=cuda)
    out = node_log_probs(x, torch.zeros_like(labels))
    (grad,) = torch.autograd.grad(out.log_prob, x, w)
    assert torch.isfinite(grad).all() and not grad[1:].any()


def test_sure_rows_keep_their_digits(cuda):
    """One class with nearly all of the probability: log p and H are small, not 0."""
    for c in (3, 60, 700, 30000):
        x = torch.zeros(2, c, device=cuda)
        x[:, 1] = torch.tensor([25.0, 14.0], device=cuda)
        labels = torch.ones(2, dtype=torch.int64, device=cuda)
        x.requires_grad_()
        # 1 + e^-25 keeps 16 - 11 digits of the small term in 64 bits, so the oracle takes log1p of the small sum:
        # s = (c - 1) e^-d, log p = -log1p(s), H = log1p(s) + d s / (1 + s)
        d = x.detach()[:, 1].double()
        s = (c - 1) * torch.exp(-d)
        lp, H = -torch.log1p(s), torch.log1p(s) + d * s / (1 + s)
        p = (torch.exp(-d) / (1 + s))[:, None].expand(2, c)
        out = node_log_probs(x, labels)
        check(out.log_prob, lp, 64 * U * lp.abs(), "log_prob")
        check(out.entropy, H, 64 * U * H, "entropy")
        (grad,) = torch.autograd.grad(out.log_prob.sum(), x)
        want = -p.clone()
        want[:, 1] = -torch.expm1(lp)
        check(grad, want, 64 * U * want.abs(), "grad")


def test_broadcast_gradient_and_single_outputs(cuda):
    x, labels, _ = make(cuda, 300, 47, torch.float32)
    x.requires_grad_()
    out = node_log_probs(x, labels, 3)
    assert isinstance(out, NodeLogProbs)
    ones = torch.ones(300, device=cuda)
    for one in (out.log_prob, out.entropy):
        (a,) = torch.autograd.grad(one.sum(), x, retain_graph=True)       # an expanded scalar
        (b,) = torch.autograd.grad(one, x, ones, retain_graph=True)
        assert torch.equal(a, b)
    (a,) = torch.autograd.grad(out.top_log_probs.sum(), x, retain_graph=True)
    (b,) = torch.autograd.grad(out.top_log_probs, x, torch.ones(3, 300, device=cuda).t(), retain_graph=True)
    assert torch.equal(a, b)
    wide = torch.zeros(300, 4, device=cuda)
    wide[:, 1] = 1
    (a,) = torch.autograd.grad(out.log_prob, x, wide[:, 1], retain_graph=True)  # a strided gradient
    (b,) = torch.autograd.grad(out.log_prob, x, ones)
    assert torch.equal(a, b)


def test_equals_cross_entropy_on_the_labelled_rows(cuda):
    x, labels, _ = make(cuda, 2000, 5, torch.float32, "padded")
    x.requires_grad_()
    lp = node_log_probs(x, labels).log_prob
    count = (labels >= 0).sum()
    (grad,) = torch.autograd.grad(-lp.sum() / count, x)
    xr = x.detach().double().requires_grad_()
    loss = torch.nn.functional.cross_entropy(xr, labels, ignore_index=-100)
    (want,) = torch.autograd.grad(loss, xr)
    check(-lp.sum() / count, loss, 2048 * U * loss.abs().detach(), "loss")
    check(grad, want, 64 * U * want.abs(), "grad")


def test_gradient_against_differences(cuda):
    x, labels, g = make(cuda, 8, 30, torch.float32, spread=1.0)
    gl, gh = torch.randn(8, generator=g, device=cuda), torch.randn(8, generator=g, device=cuda)
    gt = torch.randn(8, 3, generator=g, device=cuda)

    def loss(t):
        o = node_log_probs(t, labels, 3)
        return o, (o.log_prob.double() * gl + o.entropy.double() * gh + (o.top_log_probs.double() * gt).sum(1)).sum()
    x.requires_grad_()
    (grad,) = torch.autograd.grad(loss(x)[1], x)
    h = 2.0 ** -6
    v = torch.randn(8, 30, generator=g, device=cuda)
    v = v / v.norm()
    up, down = loss(x.detach() + h * v), loss(x.detach() - h * v)
    assert torch.equal(up[0].top_index, down[0].top_index)
    diff = float(up[1] - down[1]) / (2 * h)
    weight = float((gl.abs() + 8 * gh.abs() + gt.abs().sum(1)).sum())
    # third derivatives of a log softmax along a unit step are at most 8
    assert abs(diff - float((grad.double() * v.double()).sum())) <= weight * (8 * h * h / 6 + 64 * U * 12 / h)


def test_empty_and_offsets(cuda):
    x = torch.zeros(0, 9, device=cuda, requires_grad=True)
    out = node_log_probs(x, torch.zeros(0, dtype=torch.int64, device=cuda), 2)
    (grad,) = torch.autograd.grad(out.log_prob.sum(), x)
    assert grad.shape == (0, 9) and out.top_index.shape == (0, 2)


def test_offsets_past_32_bits(cuda):
    """Rows more than 2^32 elements into a buffer (bf16, a row stride of 2^26)."""
    n, ld = 70, 1 << 26
    buf = torch.empty(n * ld, dtype=torch.bfloat16, device=cuda)
    for c in (5, 2000):
        x = buf.as_strided((n, c), (ld, 1))
        x.copy_(torch.randn(n, c, device=cuda))
        labels = torch.randint(0, c, (n,), device=cuda)
        a = node_log_probs(x, labels, 3)
        b = node_log_probs(x.contiguous(), labels, 3)
        for p, q in zip(a, b):
            assert torch.equal(p, q)
    del buf


def test_repeats_bit_for_bit_on_streams_and_in_graphs(cuda):
    x, labels, _ = make(cuda, 700, 1200, torch.bfloat16)
    x.requires_grad_()
    out = {}

    def step():
        o = node_log_probs(x, labels, 5)
        out["o"] = [t.detach() for t in o]
        (out["g"],) = torch.autograd.grad((o.log_prob, o.entropy), x, (torch.ones_like(o.log_prob), torch.ones_like(o.entropy)))
        return o.log_prob.detach()
    step()
    first = [t.clone() for t in (*out["o"], out["g"])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip((*out["o"], out["g"]), first):
        assert torch.equal(a, b)
    graph = GraphedStep(step, cuda, warmup=2)
    captured = [*out["o"], out["g"]]
    for _ in range(2):
        graph()
        torch.cuda.synchronize()
        for a, b in zip(captured, first):
            assert torch.equal(a, b)


def test_second_derivative_is_refused(cuda):
    x = torch.randn(4, 8, device=cuda, requires_grad=True)
    (g,) = torch.autograd.grad(node_log_probs(x).entropy.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_refusals(cuda):
    x = torch.randn(4, 8, device=cuda)
    y = torch.zeros(4, dtype=torch.int64, device=cuda)
    for args, error in (((x.double(), y), TypeError), ((x.cpu(), y), TypeError), ((x, y.int()), TypeError),
                        ((x, y.cpu()), TypeError), ((x, y[:3]), ValueError), ((x, y[:, None]), ValueError),
                        ((x[0], y), ValueError), ((x[:, :0], y), ValueError), ((x, y, 9), ValueError),
                        ((x, y, -1), ValueError), ((torch.randn(2, 100, device=cuda), None, 65), ValueError)):
        with pytest.raises(error):
            node_log_probs(*args)
