"""Helpers of the class-row operator tests (layer_norm, node_log_probs,
distill_top_logits): inputs on a given layout, and the elementwise check.

U = 2^-24 is the largest relative error of one float32 rounding.  Where a test
allows `k * U * scale`, scale is the sum of magnitudes that enter the value and
k counts the roundings on the longest way to it: a thread adds its share of
the row one after the other and the block joins 256 threads in 13 steps, so a
sum over c terms has at most c / 256 + 13 roundings, to which the few of each
term (a product, an exponential of at most 2 units) are added.  The output's
own rounding, at most eps / 2 of its type, comes on top.
"""
import torch

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def layout(t, dtype, kind):
    """t [n, c] as `dtype`: contiguous, as part of a wider buffer, or (kind
    "shifted") as contiguous rows that start one element into a buffer."""
    t = t.to(dtype)
    n, c = t.shape
    if kind == "padded":
        buf = torch.full((n, c + 3), float("nan"), dtype=dtype, device=t.device)
        buf[:, :c] = t
        return buf[:, :c]
    if kind == "shifted":
        buf = torch.full((n * c + 1,), float("nan"), dtype=dtype, device=t.device)
        buf[1:] = t.reshape(-1)
        return buf[1:].view(n, c)
    return t.contiguous()


def sum_ulps(c):
    return c / 256 + 13


def check(actual, exact, allowed, what):
    """|actual - exact| <= allowed + the output type's rounding, elementwise;
    infinities and NaN in the same places."""
    a, e = actual.detach().double(), exact.detach().double()
    assert a.shape == e.shape, (what, a.shape, e.shape)
    assert torch.equal(torch.isnan(a), torch.isnan(e)), f"{what}: NaN in other places"
    same = (a == e) | torch.isnan(e)
    u = torch.finfo(actual.dtype).eps / 2
    # below the smallest normal number the steps do not shrink any further
    tiny = torch.finfo(actual.dtype).smallest_normal * u
    err = torch.where(same, 0.0, (a - e).abs())
    room = torch.where(same, 1.0, allowed * (1 + u) + u * e.abs() + tiny)
    worst = (err / room).nan_to_num(nan=float("inf")).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} times the allowed error"
