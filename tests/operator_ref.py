"""The tensor operators' formulas in 64 bits, with a bound on how far a kernel's result may be from them.

u(t) is half a step of type t relative to the value (finfo.eps / 2); a result of that type is off by u(t) |value| from its one
rounding, and what comes before it is in 32 bits: a sum of n products is off by at most (n + 16) u(fp32) times the sum of their
magnitudes (n additions in any order, and 16 for the products themselves, the bias and the conversions)."""
import math

import numpy as np
import torch

U32 = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["none", "lrelu", "xtanh", "sigmoid", "gelu", "silu"]
SLOPE = 0.1
# bounds of |act'| and |act''| (xtanh: 1 + slope and 4 / (3 sqrt 3); gelu: 1.129 and 2 phi(0); silu: 1.1 and 1/2; sigmoid: 1/4 and 0.0963)
LIP = {"none": 1.0, "lrelu": 1.0, "xtanh": 1.1, "sigmoid": 0.25, "gelu": 1.13, "silu": 1.1}
CURV = {"none": 0.0, "lrelu": 0.0, "xtanh": 0.77, "sigmoid": 0.0963, "gelu": 0.798, "silu": 0.5}


def u(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half a step among the type's subnormal numbers."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def act64(s, act, slope=SLOPE):
    """-> (act(s), act'(s))."""
    sig = torch.special.expit(s)
    if act == "lrelu":
        k = torch.where(s > 0, 1.0, slope).to(s.dtype)
        return s * k, k
    if act == "xtanh":
        t = torch.tanh(s)
        return t + slope * s, 1 - t * t + slope
    if act == "sigmoid":
        return sig, sig * (1 - sig)
    if act == "gelu":
        cdf = torch.special.ndtr(s)
        return s * cdf, cdf + s * torch.exp(-s * s / 2) / math.sqrt(2 * math.pi)
    if act == "silu":
        return s * sig, sig * (1 + s * (1 - sig))
    return s, torch.ones_like(s)


def linear64(x, w, b, act, residual, dy=None, slope=SLOPE):
    """CPU tensors of the operator's type -> {name: (value, bound)} for y and, with dy, dx, dw, db."""
    dt = x.dtype
    X, W = x.double(), w.double()
    k, n, m = X.shape[1], W.shape[0], X.shape[0]
    s = X @ W.t()
    mag = X.abs() @ W.abs().t()
    if b is not None:
        s, mag = s + b.double(), mag + b.double().abs()
    ds_err = (k + 16) * U32 * mag
    a, slope_s = act64(s, act, slope)
    y = a if residual is None else a + residual.double()
    r = residual.double().abs() if residual is not None else 0.0
    out = {"y": (y, u(dt) * y.abs() + tiny(dt) + LIP[act] * ds_err + 8 * U32 * (a.abs() + s.abs() + r))}
    if dy is None:
        return out
    D = dy.double()
    ds = D * slope_s
    # the derivative: s is off by its sum's error and (for bf16) by its rounding to fp16; evaluating it costs 16 roundings of at most (1 + |s|)
    kept = ds_err + ((2.0 ** -11) * s.abs() + 2.0 ** -24 if dt == torch.bfloat16 else 0.0)
    # beyond fp16's range act' has reached its limit: |s| counts up to 65504
    err = D.abs() * (CURV[act] * kept + (16 * U32 * (1 + s.abs().clamp(max=100.0)) if act != "none" else 0.0))
    if act == "lrelu":
        err = err + D.abs() * abs(1 - slope) * (s.abs() <= ds_err)
    err_sum = err
    if act != "none":
        err = err + u(dt) * (ds.abs() + err) + tiny(dt)      # ds is rounded to the type before the products
    out["dx"] = (ds @ W, err @ W.abs() + (n + 16) * U32 * ((ds.abs() + err) @ W.abs()))
    out["dw"] = (ds.t() @ X, err.t() @ X.abs() + (m + 16) * U32 * ((ds.abs() + err).t() @ X.abs()))
    out["db"] = (ds.sum(0), err_sum.sum(0) + (m + 16) * U32 * ds.abs().sum(0))
    for name in ("dx", "dw", "db"):
        v, e = out[name]
        out[name] = (v, e * (1 + u(dt)) + u(dt) * v.abs() + tiny(dt))
    return out


def norm64(x, w, b, eps, dy=None, residual=None, wdtype=None):
    """-> {name: (value, bound)} for y and, with dy, dx, dw, db."""
    dt, wt = x.dtype, wdtype or x.dtype
    X = x.double()
    m, d = X.shape
    W = w.double() if w is not None else torch.ones(d, dtype=torch.float64)
    mean = X.mean(1, keepdim=True)
    c = X - mean
    var = c.square().mean(1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    xh = c * r
    y = xh * W + (b.double() if b is not None else 0.0)
    n = d + 16                                    # a sum of d values is off by at most this many roundings of the sum of magnitudes
    e_mean = n * U32 * X.abs().mean(1, keepdim=True)
    e_c = e_mean + U32 * c.abs()
    # relative error of r: half of the variance's, which is its sum's, its terms' (2 U32 and the mean's error: second order) and the root's
    e_r = 0.5 * ((n + 4) * U32 + (e_mean * r) ** 2) + 4 * U32
    e_xh = r * e_c + xh.abs() * e_r + 2 * U32 * xh.abs()
    bb = b.double().abs() if b is not None else 0.0
    out = {"y": (y, e_xh * W.abs() + 4 * U32 * (y.abs() + (xh * W).abs() + bb) + u(dt) * y.abs() + tiny(dt))}
    if dy is None:
        return out
    D = dy.double()
    a = D * W
    m1, m2 = a.mean(1, keepdim=True), (a * xh).mean(1, keepdim=True)
    e_m1 = n * U32 * a.abs().mean(1, keepdim=True)
    e_m2 = n * U32 * (a * xh).abs().mean(1, keepdim=True) + (a.abs() * e_xh).mean(1, keepdim=True)
    inner = a - m1 - xh * m2
    dx = r * inner
    e = r * (4 * U32 * (a.abs() + m1.abs() + (xh * m2).abs()) + e_m1 + e_xh * m2.abs() + (xh.abs() + e_xh) * e_m2) + (e_r + 2 * U32) * dx.abs()
    if residual is not None:
        dx = dx + residual.double()
        e = e + U32 * (dx.abs() + residual.double().abs())
    out["dx"] = (dx, e + u(dt) * dx.abs() + tiny(dt))
    dw, db = (D * xh).sum(0), D.sum(0)
    out["dw"] = (dw, (D.abs() * e_xh).sum(0) + (m + 16) * U32 * (D * xh).abs().sum(0) + u(wt) * dw.abs() + tiny(wt))
    out["db"] = (db, (m + 16) * U32 * D.abs().sum(0) + u(wt) * db.abs() + tiny(wt))
    return out


def keep(n, p, seed, offset):
    """The dropout mask of n elements, in numpy's wrapping unsigned integers."""
    U = np.uint64
    e = np.arange((n + 3) // 4, dtype=U)
    lo, h = U(0xFFFFFFFF), U(32)
    seed, offset = seed % 2 ** 64, offset % 2 ** 64
    c = [e & lo, e >> h, np.full_like(e, offset % 2 ** 32), np.full_like(e, offset >> 32)]
    k = [seed % 2 ** 32, seed >> 32]
    for _ in range(10):
        a, b = c[0] * U(0xD2511F53), c[2] * U(0xCD9E8D57)
        c = [(b >> h) ^ c[1] ^ U(k[0]), b & lo, (a >> h) ^ c[3] ^ U(k[1]), a & lo]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    words = np.stack(c, 1).reshape(-1)[:n]
    return torch.from_numpy(words >= U(int(p * 2.0 ** 32))) if p < 1 else torch.zeros(n, dtype=torch.bool)


def close(got, want, what):
    """`got` (any device) against (value, bound)."""
    value, bound = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    bad = ~((got - value).abs() <= bound)
    assert not bad.any(), (what, int(bad.sum()), "of", bad.numel(), "worst", float(((got - value).abs() / bound.clamp(min=1e-300)).max()),
                           "first at", bad.nonzero()[0].tolist())
