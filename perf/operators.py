"""The operators of a residual MLP block, in plain torch operations and as calls of this framework:

  linear      y = act(x W^T + b) + residual, and its gradients
  layer_norm  y = (x - mean) / sqrt(var + eps) * g + c over the last dimension, and its gradients
  dropout     y = keep * x / (1 - p) + residual, keep drawn by Philox4x32-10 from (seed, offset, element number)
  block       y = h + dropout(W2 act(W1 layer_norm(h) + b1) + b2), forward and backward: the three run together

`own` selects the framework's calls; the plain forms run anywhere torch does."""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
ACTS = ("none", "lrelu", "xtanh", "sigmoid", "gelu", "silu")
SLOPE = 0.1
EPS = 1e-5


def listed():
    return [
        # one token through a square projection of a model that is being served: all of it is reading the weights
        {"name": "linear_one_row_bf16", "op": "linear", "mode": "forward", "rows": 1, "inner": 4096, "outer": 4096, "dtype": "bfloat16",
         "act": "silu", "residual": True},
        # the tokens of a few requests through an MLP's first projection
        {"name": "linear_few_rows_fp16", "op": "linear", "mode": "forward", "rows": 24, "inner": 2048, "outer": 8192, "dtype": "float16",
         "act": "gelu", "residual": False},
        # a hidden layer of the default encoder (batch 64, width 50), one training step: nothing but latency
        {"name": "linear_hidden_fp32", "op": "linear", "mode": "train", "rows": 64, "inner": 50, "outer": 50, "dtype": "float32",
         "act": "lrelu", "residual": True},
        # a wide encoder's hidden layer in the framework's own type
        {"name": "linear_wide_fp32", "op": "linear", "mode": "train", "rows": 8192, "inner": 2048, "outer": 2048, "dtype": "float32",
         "act": "xtanh", "residual": True},
        # sizes that fit no tile and rows that no wide load is aligned to
        {"name": "linear_ragged_fp16", "op": "linear", "mode": "train", "rows": 1531, "inner": 1001, "outer": 777, "dtype": "float16",
         "act": "sigmoid", "residual": False},
        # the largest: a training step of an MLP projection over 8192 tokens
        {"name": "linear_large_bf16", "op": "linear", "mode": "train", "rows": 8192, "inner": 4096, "outer": 4096, "dtype": "bfloat16",
         "act": "gelu", "residual": True},
        # one token while serving
        {"name": "norm_one_row_bf16", "op": "layer_norm", "mode": "forward", "rows": 1, "inner": 4096, "dtype": "bfloat16"},
        # the norm of a training step over 16384 tokens
        {"name": "norm_large_bf16", "op": "layer_norm", "mode": "train", "rows": 16384, "inner": 4096, "dtype": "bfloat16"},
        # odd rows of odd width
        {"name": "norm_ragged_fp32", "op": "layer_norm", "mode": "train", "rows": 5003, "inner": 1037, "dtype": "float32"},
        # a hidden layer of the widest configuration here (batch 64, width 200)
        {"name": "dropout_hidden_fp32", "op": "dropout", "mode": "train", "rows": 64, "inner": 200, "dtype": "float32", "p": 0.1,
         "residual": True},
        # activations of a large training step, added to the stream they belong to
        {"name": "dropout_large_bf16", "op": "dropout", "mode": "train", "rows": 8192, "inner": 8192, "dtype": "bfloat16", "p": 0.1,
         "residual": True},
        # the three together, one training step of a residual block
        {"name": "block_fp32", "op": "block", "mode": "train", "rows": 4096, "inner": 1024, "outer": 4096, "dtype": "float32", "act": "gelu",
         "p": 0.1},
    ]


def _log_uniform(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "layer_norm", "layer_norm", "dropout", "block"])
    case = {"op": op, "mode": rng.choice(["forward", "train", "train"]), "dtype": rng.choice(sorted(DTYPES))}
    if op == "linear":
        case.update(rows=_log_uniform(rng, 1, 8192), inner=_log_uniform(rng, 16, 4096), outer=_log_uniform(rng, 16, 4096), act=rng.choice(ACTS),
                    residual=rng.random() < 0.5)
        if rng.random() < 0.4:      # sizes of real layers are round more often than not
            case.update(inner=-(-case["inner"] // 64) * 64, outer=-(-case["outer"] // 64) * 64)
    elif op == "layer_norm":
        case.update(inner=_log_uniform(rng, 16, 16384))
        case.update(rows=_log_uniform(rng, 1, 16384 * 4096 // max(4096, case["inner"])))
    elif op == "dropout":
        case.update(rows=_log_uniform(rng, 1, 8192), inner=_log_uniform(rng, 16, 8192), p=round(rng.uniform(0.0, 0.6), 3), residual=rng.random() < 0.5)
    else:
        # the activations between the operators of a block are rounded to its type: in 32 bits a block's outputs are the formula's
        case.update(mode="train", dtype="float32", rows=_log_uniform(rng, 1, 4096), inner=_log_uniform(rng, 16, 1024), outer=_log_uniform(rng, 16, 4096),
                    act=rng.choice(ACTS), p=round(rng.uniform(0.0, 0.6), 3))
    # lrelu's slope jumps at 0. Among millions of sums in 32 bits some are so near to 0 that the order of summation decides on which side they
    # land; in a large product of that type the activation is one whose slope is continuous.
    if case.get("act") == "lrelu" and case["dtype"] == "float32" and case["rows"] * case["outer"] > 1 << 16:
        case["act"] = rng.choice([a for a in ACTS if a != "lrelu"])
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------------


def prepare(case, seed):
    """Inputs of unit scale, weights of a layer's usual scale, gradients of unit scale."""
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=gen, device=dev) * scale + shift).to(dt)

    rows, inner, outer = case["rows"], case["inner"], case.get("outer", 0)
    s = {"case": dict(case), "x": normal(rows, inner)}
    if case["op"] == "linear":
        s.update(w=normal(outer, inner, scale=inner ** -0.5), b=normal(outer, scale=0.1), dy=normal(rows, outer),
                 residual=normal(rows, outer) if case["residual"] else None)
    elif case["op"] == "layer_norm":
        s.update(x=normal(rows, inner, scale=1.5, shift=0.3), g=normal(inner, scale=0.1, shift=1.0), c=normal(inner, scale=0.1), dy=normal(rows, inner))
    elif case["op"] == "dropout":
        s.update(dy=normal(rows, inner), residual=normal(rows, inner) if case["residual"] else None)
    else:
        s.update(g=normal(inner, scale=0.1, shift=1.0), c=normal(inner, scale=0.1), w1=normal(outer, inner, scale=inner ** -0.5),
                 b1=normal(outer, scale=0.1), w2=normal(inner, outer, scale=outer ** -0.5), b2=normal(inner, scale=0.1), dy=normal(rows, inner))
    s["seed"], s["offset"] = 0x9E3779B97F4A7C15 ^ int(seed), 1000003 + 7 * int(seed)
    return s


# ---- plain forms: 32 bits, rounded once at the end ------------------------------------------------------------------


def _act(s, act):
    if act == "lrelu":
        return torch.where(s > 0, s, SLOPE * s)
    if act == "xtanh":
        return torch.tanh(s) + SLOPE * s
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-s))
    if act == "gelu":
        return 0.5 * s * (1 + torch.erf(s * math.sqrt(0.5)))
    if act == "silu":
        return s / (1 + torch.exp(-s))
    return s


def _act_slope(s, act):
    """d act / d s."""
    if act == "lrelu":
        return torch.where(s > 0, 1.0, SLOPE)
    if act == "xtanh":
        return 1 - torch.tanh(s).square() + SLOPE
    if act == "sigmoid":
        t = 1 / (1 + torch.exp(-s))
        return t * (1 - t)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(s * math.sqrt(0.5))) + s * torch.exp(-0.5 * s * s) * (1 / math.sqrt(2 * math.pi))
    t = 1 / (1 + torch.exp(-s))
    return t * (1 + s * (1 - t))


def _linear(x, w, b, act):
    """-> (act(s), s), s = x w^T + b."""
    s = x @ w.t() + b
    return _act(s, act), s


def _linear_back(dy, x, w, s, act):
    """-> (dx, dw, db)."""
    ds = dy if act == "none" else dy * _act_slope(s, act)
    return ds @ w, ds.t() @ x, ds.sum(0)


def _norm(x, g, c):
    """-> (y, xhat, 1 / sqrt(var + eps))."""
    mid = x - x.mean(1, keepdim=True)
    r = torch.rsqrt(mid.square().mean(1, keepdim=True) + EPS)
    xhat = mid * r
    return xhat * g + c, xhat, r


def _norm_back(dy, xhat, r, g):
    """-> (dx, dg, dc)."""
    dxhat = dy * g
    dx = r * (dxhat - dxhat.mean(1, keepdim=True) - xhat * (dxhat * xhat).mean(1, keepdim=True))
    return dx, (dy * xhat).sum(0), dy.sum(0)


def _mulhilo(a, m):
    """High and low 32 bits of a * m, for 32-bit numbers held in int64 (a * m itself would pass 63 bits)."""
    top = (a >> 16) * m
    low = (a & 0xFFFF) * m
    return (top + (low >> 16)) >> 16, (a * m) & 0xFFFFFFFF


def _keep(shape, p, seed, offset, dev):
    """Philox4x32-10 (Salmon et al. 2011) of the counter (e // 4, offset) under the key `seed`: word e % 4 belongs to element e, which is
    kept where that word is at least p * 2^32."""
    n = math.prod(shape)
    q = torch.arange((n + 3) // 4, device=dev)
    c0, c1 = q & 0xFFFFFFFF, q >> 32
    c2, c3 = torch.full_like(q, offset & 0xFFFFFFFF), torch.full_like(q, (offset >> 32) & 0xFFFFFFFF)
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for _ in range(10):
        h0, l0 = _mulhilo(c0, 0xD2511F53)
        h1, l1 = _mulhilo(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return (torch.stack([c0, c1, c2, c3], 1).reshape(-1)[:n] >= int(p * 2 ** 32)).reshape(shape)


def _plain(s):
    case, dt = s["case"], DTYPES[s["case"]["dtype"]]
    f = {k: v.float() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    out = lambda *t: [None if v is None else v.to(dt) for v in t]  # noqa: E731
    train = case["mode"] == "train"
    if case["op"] == "linear":
        a, pre = _linear(f["x"], f["w"], f["b"], case["act"])
        y = a if f["residual"] is None else a + f["residual"]
        return out(y, *_linear_back(f["dy"], f["x"], f["w"], pre, case["act"])) if train else out(y)
    if case["op"] == "layer_norm":
        y, xhat, r = _norm(f["x"], f["g"], f["c"])
        return out(y, *_norm_back(f["dy"], xhat, r, f["g"])) if train else out(y)
    keep = _keep(f["x"].shape, case["p"], s["seed"], s["offset"], s["x"].device)
    scale = 1 / (1 - case["p"])
    if case["op"] == "dropout":
        y = torch.where(keep, f["x"] * scale, 0.0)
        y = y if f["residual"] is None else y + f["residual"]
        return out(y, torch.where(keep, f["dy"] * scale, 0.0)) if train else out(y)
    t, xhat, r = _norm(f["x"], f["g"], f["c"])
    a, pre = _linear(t, f["w1"], f["b1"], case["act"])
    o, _ = _linear(a, f["w2"], f["b2"], "none")
    y = f["x"] + torch.where(keep, o * scale, 0.0)
    do = torch.where(keep, f["dy"] * scale, 0.0)
    da, dw2, db2 = _linear_back(do, a, f["w2"], None, "none")
    dn, dw1, db1 = _linear_back(da, t, f["w1"], pre, case["act"])
    dx, dg, dc = _norm_back(dn, xhat, r, f["g"])
    return out(y, dx + f["dy"], dg, dc, dw1, db1, dw2, db2)


# ---- the framework's calls ------------------------------------------------------------------------------------------


def _ours(s):
    from ivae_amd import ops
    case = s["case"]
    train = case["mode"] == "train"
    if case["op"] == "linear":
        if not train:
            return [ops.linear(s["x"], s["w"], s["b"], case["act"], SLOPE, residual=s["residual"])]
        y, pre = ops.linear(s["x"], s["w"], s["b"], case["act"], SLOPE, residual=s["residual"], save=True)
        return [y, *ops.linear_backward(s["dy"], s["x"], s["w"], pre, case["act"], SLOPE)]
    if case["op"] == "layer_norm":
        if not train:
            return [ops.layer_norm(s["x"], s["g"], s["c"], EPS)]
        y, stats = ops.layer_norm(s["x"], s["g"], s["c"], EPS, save=True)
        return [y, *ops.layer_norm_backward(s["dy"], s["x"], stats, s["g"])]
    p, seed, offset = case["p"], s["seed"], s["offset"]
    if case["op"] == "dropout":
        y = ops.dropout(s["x"], p, seed, offset, residual=s["residual"])
        return [y, ops.dropout_backward(s["dy"], p, seed, offset)] if train else [y]
    t, stats = ops.layer_norm(s["x"], s["g"], s["c"], EPS, save=True)
    a, pre = ops.linear(t, s["w1"], s["b1"], case["act"], SLOPE, save=True)
    y = ops.dropout(ops.linear(a, s["w2"], s["b2"]), p, seed, offset, residual=s["x"])
    do = ops.dropout_backward(s["dy"], p, seed, offset)
    da, dw2, db2 = ops.linear_backward(do, a, s["w2"])
    dn, dw1, db1 = ops.linear_backward(da, t, s["w1"], pre, case["act"], SLOPE)
    dx, dg, dc = ops.layer_norm_backward(dn, s["x"], stats, s["g"], residual=s["dy"])
    return [y, dx, dg, dc, dw1, db1, dw2, db2]


def run(state):
    return _ours(state) if own else _plain(state)


# ---- what a pass has to do ------------------------------------------------------------------------------------------


def work(case):
    """Every input read once and every output written once; the operations of the products, or of the elements where there are none."""
    size = DTYPES[case["dtype"]].itemsize
    m, k, n, train = case["rows"], case["inner"], case.get("outer", 0), case["mode"] == "train"
    if case["op"] == "linear":
        values = m * k + n * k + n + m * n * (2 if case["residual"] else 1)
        if train:
            values += m * n + m * k + n * k + n
        return {"bytes": values * size, "flops": 2 * m * n * k * (3 if train else 1)}
    if case["op"] == "layer_norm":
        return {"bytes": (m * k * (4 if train else 2) + k * (4 if train else 2)) * size, "flops": m * k * (20 if train else 8)}
    if case["op"] == "dropout":
        return {"bytes": m * k * size * ((3 if case["residual"] else 2) + (2 if train else 0)), "flops": m * k * (4 if train else 2)}
    return {"bytes": (4 * m * k + 2 * (2 * n * k + n + 3 * k)) * size, "flops": 12 * m * n * k}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------


def _kept(n, p, seed, offset):
    """keep of n elements, with numpy's wrapping unsigned integers."""
    import numpy as np
    u = np.uint64
    e = np.arange((n + 3) // 4, dtype=u)
    low, half = u(0xFFFFFFFF), u(32)
    ctr = [e & low, e >> half, np.full_like(e, offset & 0xFFFFFFFF), np.full_like(e, offset >> 32 & 0xFFFFFFFF)]
    key = [seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF]
    for _ in range(10):
        a, b = ctr[0] * u(0xD2511F53), ctr[2] * u(0xCD9E8D57)
        ctr = [(b >> half) ^ ctr[1] ^ u(key[0]), b & low, (a >> half) ^ ctr[3] ^ u(key[1]), a & low]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    return np.stack(ctr, 1).reshape(-1)[:n] >= u(int(p * 2.0 ** 32))


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    x, dy = d["x"], d["dy"]
    act, train = case.get("act", "none"), case["mode"] == "train"

    def activation(z):
        """-> (act(z), act'(z))."""
        gate = torch.special.expit(z)
        if act == "lrelu":
            k = torch.where(z > 0, torch.ones_like(z), torch.full_like(z, SLOPE))
            return z * k, k
        if act == "xtanh":
            h = torch.tanh(z)
            return h + SLOPE * z, (1 - h) * (1 + h) + SLOPE
        if act == "sigmoid":
            return gate, gate * torch.special.expit(-z)
        if act == "gelu":
            cdf = torch.special.ndtr(z)
            return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        if act == "silu":
            return z * gate, gate + z * gate * torch.special.expit(-z)
        return z, torch.ones_like(z)

    def normalised(v):
        var, mean = torch.var_mean(v, 1, correction=0, keepdim=True)
        sd = torch.sqrt(var + EPS)
        return (v - mean) / sd, sd

    def norm_gradient(grad, hat, sd):
        w = grad * d["g"]
        return (w - w.mean(1, keepdim=True) - hat * (w * hat).mean(1, keepdim=True)) / sd, torch.einsum("rk,rk->k", grad, hat), grad.sum(0)

    if case["op"] == "linear":
        y, slope = activation(torch.addmm(d["b"], x, d["w"].t().contiguous()))
        y = y + d["residual"] if case["residual"] else y
        ds = dy * slope
        return [y, torch.mm(ds, d["w"]), torch.mm(ds.t().contiguous(), x), ds.sum(0)] if train else [y]
    if case["op"] == "layer_norm":
        hat, sd = normalised(x)
        y = hat * d["g"] + d["c"]
        return [y, *norm_gradient(dy, hat, sd)] if train else [y]
    factor = torch.from_numpy(_kept(x.numel(), case["p"], s["seed"], s["offset"])).to(x.device).reshape(x.shape).double() / (1 - case["p"])
    if case["op"] == "dropout":
        y = x * factor + (d["residual"] if case["residual"] else 0)
        return [y, dy * factor] if train else [y]
    hat, sd = normalised(x)
    t = hat * d["g"] + d["c"]
    a, slope = activation(torch.addmm(d["b1"], t, d["w1"].t().contiguous()))
    y = x + factor * torch.addmm(d["b2"], a, d["w2"].t().contiguous())
    do = dy * factor
    ds = torch.mm(do, d["w2"]) * slope
    dx, dg, dc = norm_gradient(torch.mm(ds, d["w1"]), hat, sd)
    return [y, dx + dy, dg, dc, torch.mm(ds.t().contiguous(), t), ds.sum(0), torch.mm(do.t().contiguous(), a), do.sum(0)]
