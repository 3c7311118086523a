"""Plain 64-bit forms of the training operators, with element-wise bounds on what fp32 sums and one rounding may add."""
import math

import torch

HALF = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}  # half a step, relative to the value
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134, torch.float32: 2.0**-150}  # half a step below the normal range
U = 2.0**-24  # one rounded fp32 operation


def act(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * torch.special.erfc(-z / math.sqrt(2))
    if name == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z**3))
    return z * torch.sigmoid(1.702 * z) if name == "quick_gelu" else z


def slope(z, name):
    if name in (None, "none"):
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        s = torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z**3))
        return s + z * s * (1 - s) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    a = 1.702 if name == "quick_gelu" else 1.0
    s = torch.sigmoid(a * z)
    return s + a * z * s * (1 - s)


def within(got, want, bound, what):
    """|got - want| <= bound + half a step of got's type, element by element."""
    t = got.dtype
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} is not {tuple(want.shape)}"
    off = (got.double() - want).abs()
    limit = bound + HALF[t] * (want.abs() + bound) + TINY[t]
    bad = ~(off <= limit)  # NaN counts
    # The largest finite value is (2 - 2 h) 2^e; from half a step above it on, (2 - h) 2^e, rounding gives infinity, as it has to: 60011 equal
    # rows whose value is 1.34 add up to 80463, beyond the 65520 of fp16.
    over = want.abs() + bound >= torch.finfo(t).max * (2 - HALF[t]) / (2 - 2 * HALF[t])
    bad &= ~(over & (got.double() == want.sign() * float("inf")))
    if bad.any():
        i = int((off / limit).nan_to_num(float("inf")).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off; worst at {i}: {got.flatten()[i].item()} is not "
                             f"{want.flatten()[i].item()} +- {limit.flatten()[i].item():.3g}")


def wide(t):
    return None if t is None else t.detach().double()


# ---- LayerNorm: a thread adds at most 128 values of a row (or C / 1024), then come at most 12 levels of pairwise sums
def _row_adds(c):
    return 128 + c / 1024 + 12


def norm(x, weight, bias, eps):
    """(y, its bound, mean, its bound, rstd, its bound)."""
    x, w, b = wide(x), wide(weight), wide(bias)
    c = x.shape[-1]
    k = _row_adds(c) * U
    w = torch.ones(c, dtype=x.dtype, device=x.device) if w is None else w
    b = torch.zeros(c, dtype=x.dtype, device=x.device) if b is None else b
    mean = x.mean(-1, keepdim=True)
    var = ((x - mean) ** 2).mean(-1, keepdim=True)
    rstd = 1 / (var + eps).sqrt()
    dm = k * x.abs().mean(-1, keepdim=True) + U * mean.abs()
    # a shift of the mean by dm enters the variance as dm^2 and, through rounded differences, as 2 U |x - mean|
    dvar = dm * dm + (k + 4 * U) * var + 2 * U * dm * (x - mean).abs().mean(-1, keepdim=True)
    drstd = rstd * (0.5 * dvar / (var + eps) + 4 * U)
    h = (x - mean) * rstd
    dh = rstd * (dm + U * (x - mean).abs()) + (x - mean).abs() * drstd + 2 * U * h.abs()
    y = h * w + b
    return y, w.abs() * dh + 2 * U * (h * w).abs() + U * y.abs(), mean[..., 0], dm[..., 0], rstd[..., 0], drstd[..., 0]


def norm_grad(dy, x, mean, rstd, weight):
    """(dx, bound, dweight, bound, dbias, bound) for the given mean and rstd."""
    dy, x, w = wide(dy).flatten(0, -2), wide(x).flatten(0, -2), wide(weight)
    mean, rstd = wide(mean).reshape(-1, 1), wide(rstd).reshape(-1, 1)
    rows, c = x.shape
    k = (_row_adds(c) + 4) * U
    w = torch.ones(c, dtype=x.dtype, device=x.device) if w is None else w
    h = (x - mean) * rstd
    g = dy * w
    s1, s2 = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
    d1, d2 = k * g.abs().mean(-1, keepdim=True), (k + 4 * U) * (g * h).abs().mean(-1, keepdim=True)
    dx = rstd * (g - s1 - h * s2)
    bx = rstd * (3 * U * g.abs() + 2 * U * s1.abs() + d1 + h.abs() * (d2 + 5 * U * s2.abs())) + U * dx.abs()
    # at least 64 shares of the rows (or one row each), and no more than 64 additions of shares in a row
    r = (rows / 64 + 1 + 64 + 8) * U
    dw, db = (dy * h).sum(0), dy.sum(0)
    return dx, bx, dw, (r + 4 * U) * (dy * h).abs().sum(0), db, r * dy.abs().sum(0)


# ---- linear layers: the tensor core truncates (2 U of the running sum) once for every 16 products, and adds those
# 16 in any order; 64 more operations for sums over warps and parts of the K range
def _products(k):
    return (k / 8 + 64) * 2 * U


def _act_error(z):
    # fast exponential and division, or 1 + erf where it cancels: 2^-20 of the argument and of 1
    return 2.0**-20 * (1 + z.abs())


def linear(x, weight, bias, name, residual):
    """(y, bound, pre, bound)."""
    x, w, b, r = wide(x), wide(weight), wide(bias), wide(residual)
    z = x @ w.T
    bz = _products(x.shape[-1]) * (x.abs() @ w.abs().T)
    if b is not None:
        z = z + b
        bz = bz + U * z.abs()
    y = act(z, name)
    by = 1.13 * bz + (0 if name in (None, "none", "relu") else _act_error(z))  # no slope here exceeds 1.13
    if r is not None:
        y = y + r
        by = by + U * y.abs()
    return y, by, z, bz


def linear_grad(dy, x, weight, pre, name):
    """(dx, bound, dweight, bound, dbias, bound)."""
    t = dy.dtype
    dy, x, w, pre = (None if v is None else wide(v).flatten(0, -2) for v in (dy, x, weight, pre))
    m, n = dy.shape
    plain = name in (None, "none")
    dz = dy if plain else dy * slope(pre, name)
    exactly = torch.zeros_like(dz) if plain or name == "relu" else dy.abs() * _act_error(pre)
    bz = torch.zeros_like(dz) if plain else exactly + HALF[t] * (dz.abs() + exactly) + TINY[t]
    big = dz.abs() + bz
    bx = bz @ w.abs() + _products(n) * (big @ w.abs())
    bw = bz.T @ x.abs() + _products(m) * (big.T @ x.abs())
    bb = exactly.sum(0) + (m / 8 + 1 + 8 + 160) * U * big.sum(0)
    return dz @ w, bx, dz.T @ x, bw, dz.sum(0), bb
