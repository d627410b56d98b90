"""The operators of the classification head and what they are measured on:

* layer_norm: LayerNorm of rows of any width in float32, bfloat16 or float16, and its backward pass with the
  gradients of weight and bias;
* node_log_probs: per node the log probability of its label, the entropy of its class distribution and its most
  likely classes, and the gradient of the logits;
* distill_top_logits: the divergence of a student's class distribution from a teacher's best few classes, and the
  gradient of the student's logits.

`run` computes a case in its plain form (elementary torch operations in 32 bits) or, where `own` is true, through
cign_b200; `exact` computes it from the definitions in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPS = 1e-5
DRAW_ELEMENTS = 1 << 26


# ------------------------------------------------------------------ cases
def listed():
    return [
        # the output norm of a 4-block model of width 512 on the 24,492-node graph: 5 states side by side, one training step
        dict(name="norm_jk_train", op="norm", rows=24492, cols=2560, dtype="float32", params="float32", train=True, pad=0),
        # one sampled batch of seed nodes at the model's hidden width: latency counts
        dict(name="norm_small_train", op="norm", rows=256, cols=512, dtype="float32", params="float32", train=True, pad=0),
        # a large partition's rows stored in bf16 with float32 parameters
        dict(name="norm_bf16_train", op="norm", rows=131072, cols=1024, dtype="bfloat16", params="float32", train=True, pad=0),
        # inference on raw features of an odd width (300 inputs and a degree column) stored in fp16
        dict(name="norm_fp16_odd_eval", op="norm", rows=200003, cols=301, dtype="float16", params="float16", train=False, pad=0),
        # the 5-class co-purchase graph: logits are 5 columns of rows padded to 8, half of the nodes have labels
        dict(name="logp_5_train", op="logp", rows=24492, cols=5, dtype="float32", top_k=0, labelled=0.5, train=True, pad=3),
        # the 2.45M-node graph with 47 classes, one training step
        dict(name="logp_47_train", op="logp", rows=2450000, cols=47, dtype="float32", top_k=0, labelled=0.5, train=True, pad=1),
        # evaluation over a large odd label space with 20 alternatives of each node
        dict(name="logp_wide_eval", op="logp", rows=2048, cols=65537, dtype="bfloat16", top_k=20, labelled=1.0, train=False, pad=0),
        # an online query: three nodes, a hundred thousand labels
        dict(name="logp_query_eval", op="logp", rows=3, cols=100003, dtype="float32", top_k=8, labelled=1.0, train=False, pad=0),
        # a student of the 47-class model: 5 of the teacher's classes of each node are kept
        dict(name="distill_47_train", op="distill", rows=169343, cols=47, dtype="float32", top_k=5, temperature=2.0, tail="drop", train=True, pad=1),
        # a wide label space, 64 kept classes and the rest as one class
        dict(name="distill_wide_train", op="distill", rows=4096, cols=32768, dtype="bfloat16", top_k=64, temperature=1.0, tail="bucket", train=True, pad=0),
        # a sampled batch, an odd number of labels in fp16
        dict(name="distill_odd_train", op="distill", rows=777, cols=10007, dtype="float16", top_k=20, temperature=3.0, tail="drop", train=True, pad=0),
        # the loss of a few held-out nodes: latency counts
        dict(name="distill_small_eval", op="distill", rows=16, cols=1000, dtype="float32", top_k=8, temperature=2.0, tail="bucket", train=False, pad=0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "logp", "distill"])
    dtype = rng.choice(sorted(DTYPES))
    train = rng.random() < 0.6
    pad = rng.choice([0, 0, 0, 1, 3, 8])
    cols = _log_int(rng, 8, 16384) if op == "norm" else _log_int(rng, 2, 131072)
    if rng.random() < 0.4 and cols >= 16:
        cols -= cols % 8
    rows = _log_int(rng, 1, max(1, min(2000000, DRAW_ELEMENTS // (cols + pad))))
    case = dict(op=op, rows=rows, cols=cols, dtype=dtype, train=train, pad=pad)
    if op == "norm":
        case["params"] = rng.choice(["float32", dtype])
    elif op == "logp":
        case["top_k"] = 0 if train else min(cols, rng.choice([0, 1, 5, 20, 64]))
        case["labelled"] = rng.choice([0.5, 1.0])
    else:
        case["top_k"] = min(cols, rng.choice([1, 4, 5, 16, 20, 64, 100]))
        case["temperature"] = rng.choice([1.0, 2.0, 3.0])
        case["tail"] = rng.choice(["drop", "bucket"])
    return case


# ------------------------------------------------------------------ inputs
def _rows_of(t, pad, dtype):
    """t as a [rows, cols] view of rows that are `pad` elements longer."""
    if pad == 0:
        return t.to(dtype)
    rows, cols = t.shape
    buf = torch.zeros((rows, cols + pad), dtype=dtype, device=t.device)
    buf[:, :cols] = t
    return buf[:, :cols]


def _logits(case, g, dev):
    """Logits of a trained classifier: a spread of 2 and one class of each row that stands out."""
    rows, cols = case["rows"], case["cols"]
    x = torch.randn((rows, cols), generator=g, device=dev).mul_(2.0)
    best = torch.randint(0, cols, (rows, 1), generator=g, device=dev)
    lead = 2.0 * math.log(cols) * torch.rand((rows, 1), generator=g, device=dev)
    return x.scatter_add_(1, best, lead), best.squeeze(1)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    rows, cols, dtype = case["rows"], case["cols"], DTYPES[case["dtype"]]
    st = dict(case=case)
    if case["op"] == "norm":
        scale = 0.5 + torch.rand((rows, 1), generator=g, device=dev)
        x = torch.randn((rows, cols), generator=g, device=dev).mul_(scale).add_(0.3)
        st["x"] = _rows_of(x, case["pad"], dtype)
        params = DTYPES[case["params"]]
        st["weight"] = (1.0 + 0.1 * torch.randn(cols, generator=g, device=dev)).to(params)
        st["bias"] = (0.1 * torch.randn(cols, generator=g, device=dev)).to(params)
        if case["train"]:
            st["grad_y"] = torch.randn((rows, cols), generator=g, device=dev).to(dtype)
            for name in ("x", "weight", "bias"):
                st[name] = st[name].detach().requires_grad_()
        return st
    x, best = _logits(case, g, dev)
    st["logits"] = _rows_of(x, case["pad"], dtype)
    if case["op"] == "logp":
        other = torch.randint(0, cols, (rows,), generator=g, device=dev)
        labels = torch.where(torch.rand(rows, generator=g, device=dev) < 0.7, best, other)
        if case["labelled"] < 1.0:  # nodes without a label carry -1
            labels = torch.where(torch.rand(rows, generator=g, device=dev) < case["labelled"], labels, torch.full_like(labels, -1))
        st["labels"] = labels
        if case["train"]:  # class-balancing weights of the nodes, an entropy bonus
            st["grad_log_prob"] = -(0.5 + torch.rand(rows, generator=g, device=dev))
            st["grad_entropy"] = -0.05 * torch.rand(rows, generator=g, device=dev)
    else:
        k, temp = case["top_k"], case["temperature"]
        values = torch.empty((rows, k), device=dev)
        index = torch.empty((rows, k), dtype=torch.int64, device=dev)
        step = max(1, (1 << 26) // cols)
        for r in range(0, rows, step):  # the teacher: near the student, at the kept classes
            t = x[r:r + step] + torch.randn(x[r:r + step].shape, generator=g, device=dev)
            if case["tail"] == "bucket":  # log probabilities at the temperature
                t = torch.log_softmax(t.div_(temp), dim=1)
            values[r:r + step], index[r:r + step] = torch.topk(t, k, dim=1)
        st["values"], st["index"] = values, index
        if case["train"]:
            st["grad_loss"] = 0.5 + torch.rand(rows, generator=g, device=dev)
    if case["train"]:
        st["logits"] = st["logits"].detach().requires_grad_()
    return st


# ------------------------------------------------------------------ one pass
def run(st):
    op = st["case"]["op"]
    if own:
        return {"norm": _own_norm, "logp": _own_logp, "distill": _own_distill}[op](st)
    with torch.no_grad():
        return {"norm": _plain_norm, "logp": _plain_logp, "distill": _plain_distill}[op](st)


def _own_norm(st):
    from cign_b200.layer_norm import layer_norm
    y = layer_norm(st["x"], st["weight"], st["bias"], EPS)
    if not st["case"]["train"]:
        return (y,)
    grads = torch.autograd.grad(y, (st["x"], st["weight"], st["bias"]), st["grad_y"])
    return (y.detach(), *grads)


def _own_logp(st):
    from cign_b200.node_log_probs import node_log_probs
    out = node_log_probs(st["logits"], st["labels"], st["case"]["top_k"])
    if st["case"]["train"]:
        (grad,) = torch.autograd.grad((out.log_prob, out.entropy), (st["logits"],), (st["grad_log_prob"], st["grad_entropy"]))
        return out.log_prob.detach(), out.entropy.detach(), grad
    if st["case"]["top_k"]:
        return out.log_prob, out.entropy, out.top_log_probs, out.top_index
    return out.log_prob, out.entropy


def _own_distill(st):
    from cign_b200.distill import distill_top_logits
    c = st["case"]
    loss = distill_top_logits(st["logits"], st["values"], st["index"], c["temperature"], c["tail"])
    if not c["train"]:
        return (loss,)
    (grad,) = torch.autograd.grad(loss, (st["logits"],), st["grad_loss"])
    return loss.detach(), grad


def _plain_norm(st):
    dtype = st["x"].dtype
    x, w, b = st["x"].float(), st["weight"].float(), st["bias"].float()
    xc = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((xc * xc).mean(1, keepdim=True) + EPS)
    xhat = xc * rstd
    y = (xhat * w + b).to(dtype)
    if not st["case"]["train"]:
        return (y,)
    g = st["grad_y"].float()
    gw = g * w
    gx = rstd * (gw - gw.mean(1, keepdim=True) - xhat * (gw * xhat).mean(1, keepdim=True))
    return y, gx.to(dtype), (g * xhat).sum(0).to(st["weight"].dtype), g.sum(0).to(st["bias"].dtype)


def _log_softmax(z):
    """z - log(sum exp z) of each row, in 64 bits from the sum on: of a class that nearly has all of the probability
    the logarithm is a small difference from 0."""
    d = z - z.amax(1, keepdim=True)
    return d.double() - torch.log(torch.exp(d).sum(1, keepdim=True, dtype=torch.float64))


def _plain_logp(st):
    x, labels, k = st["logits"].float(), st["labels"], st["case"]["top_k"]
    logp64 = _log_softmax(x)
    logp = logp64.float()
    p = torch.exp(logp)
    has = labels >= 0
    at = labels.clamp(min=0).unsqueeze(1)
    log_prob = torch.where(has, logp.gather(1, at).squeeze(1), 0.0)
    entropy = -(p * logp).sum(1)
    if st["case"]["train"]:
        g = torch.where(has, st["grad_log_prob"], 0.0).unsqueeze(1)
        spread = st["grad_entropy"].unsqueeze(1) * p * (logp + entropy.unsqueeze(1))
        grad = -p * g - spread
        # at the label 1 - p, without the loss of digits where p is near 1
        grad.scatter_(1, at, -torch.expm1(logp.gather(1, at)) * g - spread.gather(1, at))
        return log_prob, entropy, grad.to(st["logits"].dtype)
    if k:  # ties go to the lower class
        _, index = torch.sort(x, dim=1, descending=True, stable=True)
        index = index[:, :k].contiguous()
        return log_prob, entropy, logp.gather(1, index), index
    return log_prob, entropy


def _plain_distill(st):
    c = st["case"]
    temp, bucket = c["temperature"], c["tail"] == "bucket"
    index = st["index"]
    # the divergence of two near distributions is a small difference of sums: 64 bits up to the loss
    z = st["logits"].double() / temp
    logp = z - z.amax(1, keepdim=True)
    logp = logp - torch.log(torch.exp(logp).sum(1, keepdim=True))
    at = logp.gather(1, index)
    v = st["values"].double()
    if not bucket:
        v = v / temp
        v = v - v.amax(1, keepdim=True)
        v = v - torch.log(torch.exp(v).sum(1, keepdim=True))
    q = torch.exp(v)
    loss = (q * (v - at)).sum(1)
    mass = q.sum(1)
    p = torch.exp(logp)
    spread = mass  # what p is multiplied with outside the kept classes
    if bucket and c["top_k"] < c["cols"]:
        p_rest = p.scatter(1, index, 0.0).sum(1)
        r = (1.0 - mass).clamp(min=0.0)
        some = r > 0
        loss = loss + torch.where(some, r * (torch.log(r) - torch.log(p_rest)), 0.0)
        mass = mass + r
        spread = mass - torch.where(some, r / p_rest, 0.0)
    loss = (loss * (temp * temp)).float()
    if not c["train"]:
        return (loss,)
    grad = (p * spread.unsqueeze(1)).scatter_(1, index, mass.unsqueeze(1) * p.gather(1, index) - q)
    return loss, (grad.float() * (temp * st["grad_loss"].unsqueeze(1))).to(st["logits"].dtype)


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    step = max(1, (1 << 25) // case["cols"])  # rows at a time
    parts = []
    with torch.no_grad():
        for r in range(0, case["rows"], step):
            parts.append(_EXACT[case["op"]](st, slice(r, r + step)))
    joined = []
    for name, column in zip(_NAMES[case["op"]], zip(*parts)):
        joined.append(sum(column) if name == "sum" else torch.cat(column))
    return tuple(joined)


_NAMES = {"norm": ("rows", "rows", "sum", "sum"), "logp": ("rows",) * 4, "distill": ("rows",) * 2}


def _exact_norm(st, at):
    x, w, b = st["x"][at].double(), st["weight"].double(), st["bias"].double()
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    s = torch.sqrt(var + EPS)
    n = (x - mean) / s
    y = torch.addcmul(b, n, w)
    if not st["case"]["train"]:
        return (y,)
    g = st["grad_y"][at].double()
    d = g * w  # the gradient of n; dx = (d - <d> - n <d n>) / s
    along = torch.einsum("rc,rc->r", d, n).div(x.size(1)).unsqueeze(1)
    return y, (d - d.mean(1, keepdim=True) - n * along) / s, torch.einsum("rc,rc->c", g, n), g.sum(0)


def _exact_logp(st, at):
    x, labels = st["logits"][at].double(), st["labels"][at]
    logp = torch.log_softmax(x, dim=1)
    p = logp.exp()
    rows = torch.arange(x.size(0), device=x.device)
    known = labels != -1
    hit = torch.zeros_like(x)
    hit[rows[known], labels[known]] = 1.0
    log_prob = (hit * logp).sum(1)
    entropy = -torch.einsum("rc,rc->r", p, logp)
    if st["case"]["train"]:
        gl = st["grad_log_prob"][at].double().unsqueeze(1)
        ge = st["grad_entropy"][at].double().unsqueeze(1)
        grad = gl * (hit - p * known.unsqueeze(1)) - ge * p * (logp + entropy.unsqueeze(1))
        return log_prob, entropy, grad
    k = st["case"]["top_k"]
    if not k:
        return log_prob, entropy
    order = torch.argsort(-x, dim=1, stable=True)[:, :k]
    return log_prob, entropy, logp.gather(1, order), order


def _exact_distill(st, at):
    c = st["case"]
    temp = c["temperature"]
    x, index = st["logits"][at].double() / temp, st["index"][at]
    logp = torch.log_softmax(x, dim=1)
    v = st["values"][at].double()
    if c["tail"] == "drop":
        v = torch.log_softmax(v / temp, dim=1)
    q = v.exp()
    # the teacher over all classes: q at its kept ones; the rest's mass is spread as the student spreads it
    target = torch.zeros_like(logp).scatter_(1, index, q)
    loss = (q * (v - logp.gather(1, index))).sum(1)
    mass = q.sum(1, keepdim=True)
    if c["tail"] == "bucket" and c["top_k"] < c["cols"]:
        outside = torch.ones_like(logp, dtype=torch.bool).scatter_(1, index, False)
        log_rest = torch.logsumexp(logp.masked_fill(~outside, -math.inf), dim=1, keepdim=True)
        r = (1.0 - mass).clamp(min=0.0)
        loss = loss + (torch.xlogy(r, r) - r * log_rest).squeeze(1)
        target = target + torch.where(outside, r * (logp - log_rest).exp(), 0.0)
        mass = mass + r
    loss = loss * temp ** 2
    if not c["train"]:
        return (loss,)
    return loss, temp * st["grad_loss"][at].double().unsqueeze(1) * (mass * logp.exp() - target)


_EXACT = {"norm": _exact_norm, "logp": _exact_logp, "distill": _exact_distill}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    """Bytes: each input read once, each output written once.  Flops: the arithmetic of the formulas, an
    exponential counted as one."""
    n, c = case["rows"], case["cols"]
    size = 4 if case["dtype"] == "float32" else 2
    train = case["train"]
    if case["op"] == "norm":
        psize = 4 if case["params"] == "float32" else 2
        moved = 2 * n * c * size + 2 * c * psize
        flops = 8 * n * c
        if train:
            moved += 2 * n * c * size + 2 * c * psize
            flops += 14 * n * c
        return {"bytes": moved, "flops": flops}
    k = case["top_k"]
    if case["op"] == "logp":
        moved = n * c * size + n * 8 + n * 8 + n * k * 12
        flops = 5 * n * c
        if train:
            moved += n * c * size + n * 8
            flops += 7 * n * c
        return {"bytes": moved, "flops": flops}
    moved = n * c * size + n * k * 12 + n * 4
    flops = 4 * n * c + 6 * n * k
    if train:
        moved += n * c * size + n * 4
        flops += 5 * n * c + 3 * n * k
    return {"bytes": moved, "flops": flops}
