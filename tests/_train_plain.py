"""Float64 evaluation of the training operators' formulas, with the bounds that the
kernels' float32 arithmetic and the rounding of each output have to stay within.

A rounding to a type is off by at most half a step, eps / 2 relative (below the
normal range half the smallest step); a float32 sum of m terms in any order is off by
at most m 2^-24 of the sum of their magnitudes.  Every function returns the values
and a bound on |result - value|, element by element."""

import math

import torch

U32 = 2.0 ** -24
SMALLEST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def rounding(value, dtype):
    return value.abs() * (torch.finfo(dtype).eps / 2) + SMALLEST[dtype] / 2


def check(got, value, bound, dtype, what=""):
    """got (of `dtype`) is within bound, plus its own rounding, of value."""
    assert got.dtype is dtype and tuple(got.shape) == tuple(value.shape), (what, got.dtype, got.shape, value.shape)
    got = got.to(value.device).double()
    exact = torch.isfinite(value)
    assert torch.equal(torch.isfinite(got), exact), f"{what}: finite in other places"
    assert torch.equal(torch.isnan(got), torch.isnan(value)), f"{what}: NaN in other places"
    odd = ~exact & ~torch.isnan(value)
    assert torch.equal(got[odd], value[odd]), f"{what}: infinities differ"
    # the rounding acts on the computed value, which is itself within bound of `value`
    limit = bound * (1 + torch.finfo(dtype).eps) + rounding(value, dtype)
    excess = ((got - value).abs() - limit)[exact]
    assert excess.numel() == 0 or float(excess.max()) <= 0, f"{what}: {float(excess.max()):.3e} over the bound"


def gather(weight, tokens, scale, row0, dtype):
    at = tokens.long() - row0
    inside = (at >= 0) & (at < weight.shape[0])
    value = torch.zeros(*tokens.shape, weight.shape[1], dtype=torch.float64, device=weight.device)
    value[inside] = weight[at[inside]].double() * scale
    return value, value.abs() * 3 * U32  # scale to float32, the product


def embedding_grad(grad, tokens, rows, scale, row0=0, padding=None, into=None):
    at = tokens.long().reshape(-1) - row0
    inside = (at >= 0) & (at < rows)
    if padding is not None:
        inside &= tokens.reshape(-1) != padding
    g = grad.reshape(-1, grad.shape[-1])[inside].double()
    at = at[inside]
    value = torch.zeros(rows, grad.shape[-1], dtype=torch.float64, device=grad.device)
    size = value.clone()
    value.index_add_(0, at, g)
    size.index_add_(0, at, g.abs())
    count = torch.zeros(rows, dtype=torch.float64, device=grad.device)
    count.index_add_(0, at, torch.ones_like(at, dtype=torch.float64))
    value, size = value * scale, size * abs(scale)
    bound = size * (count[:, None] + 3) * U32
    if into is not None:
        value = value + into.double()
        bound = bound + (size + into.double().abs()) * U32
    return value, bound


def _rsqrt_mean(v, eps):
    return torch.rsqrt(v.square().mean(-1, keepdim=True) + eps)


def block_norm(residual, x, post, pre, gate, scale, eps):
    """(h, its bound), (y, its bound); y None without pre."""
    wide = lambda t: None if t is None else t.double()  # noqa: E731
    residual, x, post, pre, gate = map(wide, (residual, x, post, pre, gate))
    c = (residual.shape[-1] + 32) * U32  # relative error of a mean of squares and the products behind it
    h, size = residual, residual.abs()
    if x is not None:
        p = x if post is None else x * _rsqrt_mean(x, eps) * post
        p = scale * p if gate is None else scale * p * gate
        h, size = h + p, size + p.abs()
    if pre is None:
        return (h, size * c), None
    r = _rsqrt_mean(h, eps)
    # the error of h relative to its row's size moves the mean of squares as well
    moved = (size * h.abs()).mean(-1, keepdim=True) * r.square()
    return (h, size * c), (h * r * pre, (size + h.abs() * (1 + moved)) * r * pre.abs() * 2 * c)


def block_norm_grad(h, x, dh, dy, post, pre, gate, scale, eps):
    """Five (value, bound) pairs or None: d_residual, d_x, d_post, d_pre, d_gate."""
    wide = lambda t: None if t is None else t.double()  # noqa: E731
    shape = h.shape
    gate_shape = None if gate is None else gate.shape
    h, x, dh, dy, post, pre, gate = map(wide, (h, x, dh, dy, post, pre, gate))
    d = shape[-1]
    rows = h.numel() // d
    c = (d + 32) * U32
    mean = lambda v: v.mean(-1, keepdim=True)  # noqa: E731
    rh = _rsqrt_mean(h, eps)
    n = h * rh
    e, size = (torch.zeros_like(h), torch.zeros_like(h)) if dh is None else (dh, dh.abs())
    d_pre = None
    if dy is not None:
        dn = dy * pre
        e = e + rh * (dn - n * mean(dn * n))
        size = size + rh * (dn.abs() + n.abs() * mean((dn * n).abs()))
        t = (dy * n).reshape(-1, d)
        d_pre = (t.sum(0), t.abs().sum(0) * (rows * U32 + 2 * c))
    d_res = (e, size * 4 * c)
    if x is None:
        return d_res, None, None, d_pre, None
    q = x if post is None else x * _rsqrt_mean(x, eps)
    w = torch.ones_like(h[..., :1]) if post is None else post
    g = torch.ones_like(h[..., :1]) if gate is None else gate
    dq = scale * e * g * w
    size_q = abs(scale) * size * g.abs() * w.abs()
    if post is None:
        d_x, d_post = (dq, size_q * 5 * c), None
    else:
        rx = _rsqrt_mean(x, eps)
        d_x = (rx * (dq - q * mean(dq * q)), rx * (size_q + q.abs() * mean(size_q * q.abs())) * 8 * c)
        t, s = (scale * e * g * q).reshape(-1, d), (scale * size * g * q).abs().reshape(-1, d)
        d_post = (t.sum(0), s.sum(0) * (rows * U32 + 6 * c))
    d_gate = None
    if gate is not None:
        full, s = scale * e * q * w, (scale * size * q * w).abs()
        lead = (1,) * (len(shape) - len(gate_shape)) + tuple(gate_shape)
        over = [i for i in range(len(shape) - 1) if lead[i] == 1 and shape[i] != 1]
        if over:
            full, s = full.sum(over, keepdim=True), s.sum(over, keepdim=True)
        d_gate = (full.reshape(gate_shape), s.reshape(gate_shape) * (rows * U32 + 6 * c))
    return d_res, d_x, d_post, d_pre, d_gate


def distill(logits, ids, teacher, weight, tau):
    """(loss, its bound), (gradient, its bound) over rows (n, vocab)."""
    vocab = logits.shape[-1]
    z = logits.double() / tau
    n, k = ids.shape
    ids = ids.long()
    w = torch.ones(n, dtype=torch.float64, device=z.device) if weight is None else weight.double()
    u = teacher.double() / tau
    valid = (ids >= 0) & (ids < vocab) & ~torch.isneginf(u)
    live = (w != 0) & valid.any(1)
    u = torch.where(valid, u, -math.inf)
    um = torch.where(live[:, None], u.amax(1, keepdim=True), 0.0) if k else torch.zeros(n, 1, dtype=z.dtype, device=z.device)
    s = torch.exp(u - um).sum(1, keepdim=True)
    p = torch.where(valid, torch.exp(u - um) / s, 0.0)
    log_p = torch.where(valid, u - um - s.log(), 0.0)
    m = z.amax(1, keepdim=True)
    m = torch.where(torch.isneginf(m), 0.0, m)
    e = torch.exp(z - m)
    norm = e.sum(1, keepdim=True)
    dead = norm == 0  # a row of -inf alone: q = 0
    q = torch.where(dead, 0.0, e / norm)
    log_q = z - m - torch.where(dead, 0.0, norm.log())
    at = ids.clamp(0, vocab - 1)
    lq = log_q.gather(1, at)
    term = torch.where(p == 0, 0.0, p * (log_p - lq))
    loss = torch.where(live, w * tau ** 2 * term.sum(1), 0.0)
    target = torch.zeros_like(z).scatter_add_(1, at, p)
    grad = torch.where(live[:, None], (w * tau)[:, None] * (q - target), 0.0)
    # exponents are off by a few roundings of their terms, sums by their length
    reach = lambda v: torch.where(torch.isfinite(v), v.abs(), 0.0).amax(1) if v.shape[1] else torch.zeros(n, dtype=z.dtype, device=z.device)  # noqa: E731
    dq = (8 * reach(z) + vocab + 64) * U32
    dp = (8 * reach(torch.where(valid, teacher.double() / tau, 0.0)) + k + 64) * U32
    size = torch.where(torch.isfinite(term), term.abs(), 0.0).sum(1)
    wide = torch.where(torch.isfinite(w), w.abs(), 0.0)
    loss_bound = wide * tau ** 2 * (size * (2 * dp + (k + 8) * U32) + dq + dp)
    grad_bound = (wide * tau)[:, None] * (torch.nan_to_num(q) * dq[:, None] + torch.nan_to_num(target) * dp[:, None])
    # an exponential below the normal range, 2^-126, may count as zero: relative to a sum of at least
    # 0.5 its q is off by at most 2^-125
    flushed = (wide * tau)[:, None] * 2.0 ** -125
    return (loss, loss_bound), (grad, 2 * grad_bound + flushed)
