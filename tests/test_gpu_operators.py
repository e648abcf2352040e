"""linear, layer_norm and dropout against their formulas in 64 bits (tests/operator_ref.py derives the bounds), forward and backward."""
import pytest
import torch

from ivae_amd import MLP, ops
from tests import operator_ref as R

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def dev():
    return torch.device("cuda:0")


def normal(g, *shape, scale=1.0, dtype=F32):
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def on(t, layout="dense"):
    """t on the GPU; `layout` places the same values at other strides or alignments (the bytes around them are NaN)."""
    if t is None:
        return None
    if layout == "dense" or t.dim() != 2:
        return t.to(dev())
    r, c = t.shape
    if layout == "strided":                         # rows of a wider matrix, at an odd offset
        big = torch.full((r, c + 13), float("nan"), dtype=t.dtype, device=dev())
        big[:, 5:5 + c] = t.to(dev())
        return big[:, 5:5 + c]
    if layout == "transposed":
        return t.t().contiguous().to(dev()).t()
    raise AssertionError(layout)


def run_linear(dt, m, k, n, act, res=True, bias=True, layout="dense", seed=0, need=(True, True, True)):
    g = torch.Generator().manual_seed(seed)
    x, w = normal(g, m, k, dtype=dt), normal(g, n, k, scale=k ** -0.5, dtype=dt)
    b = normal(g, n, scale=.3, dtype=dt) if bias else None
    r = normal(g, m, n, dtype=dt) if res else None
    dy = normal(g, m, n, dtype=dt)
    want = R.linear64(x, w, b, act, r, dy)
    X, W, B, Rr, D = on(x, layout), on(w, layout if layout != "strided" else "dense"), on(b), on(r, layout), on(dy, layout)
    y = ops.linear(X, W, B, act, R.SLOPE, residual=Rr)
    R.close(y, want["y"], "y")
    y2, saved = ops.linear(X, W, B, act, R.SLOPE, residual=Rr, save=True)
    assert torch.equal(y, y2) or torch.isnan(y).any()
    assert (saved is None) == (act == "none")
    got = ops.linear_backward(D, X, W, saved, act, R.SLOPE, need=need)
    for name, t, wanted in zip(("dx", "dw", "db"), got, need):
        if wanted:
            assert t.dtype == dt
            R.close(t, want[name], name)
        else:
            assert t is None
    return X, W, B, Rr, D, saved, y, got


SIZES = [(1, 1, 1), (1, 50, 7), (3, 16, 64), (64, 50, 50), (65, 64, 63), (7, 129, 33), (200, 33, 1), (1, 1024, 300), (2, 512, 16), (130, 257, 131),
         (17, 320, 192), (33, 96, 264), (300, 8, 8), (1000, 20, 3)]


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("dt", R.DTYPES)
def test_linear_sizes(dt, m, k, n):
    run_linear(dt, m, k, n, "gelu", seed=m + k + n)


@pytest.mark.parametrize("act", R.ACTS)
@pytest.mark.parametrize("dt", R.DTYPES)
def test_linear_activations(dt, act):
    run_linear(dt, 70, 90, 77, act, res=False, seed=3)
    run_linear(dt, 70, 96, 80, act, bias=False, seed=4)


@pytest.mark.parametrize("layout", ["strided", "transposed"])
@pytest.mark.parametrize("dt", R.DTYPES)
def test_linear_layouts(dt, layout):
    run_linear(dt, 67, 81, 35, "silu", layout=layout, seed=5)
    run_linear(dt, 64, 128, 64, "none", layout=layout, seed=6)


@pytest.mark.parametrize("need", [(True, False, False), (False, True, False), (False, False, True), (False, True, True), (True, False, True),
                                  (False, False, False)])
def test_linear_backward_parts(need):
    full = run_linear(F32, 40, 30, 20, "xtanh", seed=7)
    part = run_linear(F32, 40, 30, 20, "xtanh", seed=7, need=need)
    for a, b in zip(full[-1], part[-1]):
        assert b is None or torch.equal(a, b)


# (rows, in, out): one reduction long enough to be split, for each of the products
@pytest.mark.parametrize("m,k,n", [(3, 5000, 20), (9, 20, 5000), (6000, 17, 19), (4100, 64, 64)])
@pytest.mark.parametrize("dt", R.DTYPES)
def test_linear_long_sums(dt, m, k, n):
    run_linear(dt, m, k, n, "gelu", seed=m)


# large products: whole tiles, ragged in every direction, summed dimensions that end inside a step, few tiles with long sums
BIG = [(1024, 512, 512), (520, 768, 648), (777, 1001, 531), (64, 4104, 1000), (4100, 64, 1024), (1030, 1024, 264), (70, 72, 60000), (70, 60000, 72), (2050, 520, 1100),
       (2048, 1100, 1200), (300, 4104, 2100), (4100, 264, 2600), (6000, 264, 1000)]


@pytest.mark.parametrize("m,k,n", BIG)
@pytest.mark.parametrize("dt", R.DTYPES)
def test_linear_large(dt, m, k, n):
    run_linear(dt, m, k, n, "gelu", seed=m + 1)


@pytest.mark.parametrize("m,k,n", SIZES + BIG + [(64, 60000, 256), (4096, 200, 264), (8200, 1032, 136), (8192, 512, 4096), (3000, 2000, 2001),
                                                       (256, 4096, 8200), (20000, 256, 200), (24, 264, 8200), (50, 72, 8195), (2500, 2500, 2500), (8192, 1024, 1024)])
@pytest.mark.parametrize("dt", R.DTYPES)
def test_linear_integers_are_exact(dt, m, k, n):
    """Small whole numbers: every product and sum is one too, below 2^24, so each result is the exact one, rounded once to its type."""
    g = torch.Generator().manual_seed(m + k + n)
    x, w, dy, r = (torch.randint(-3, 4, s, generator=g).to(dt).to(dev()) for s in ((m, k), (n, k), (m, n), (m, n)))
    b = torch.randint(-9, 10, (n,), generator=g).to(dt).to(dev())
    X, W, D = x.double(), w.double(), dy.double()
    assert torch.equal(ops.linear(x, w, b, residual=r), (X @ W.t() + b.double() + r.double()).to(dt))
    for got, want in zip(ops.linear_backward(dy, x, w), (D @ W, D.t() @ X, D.sum(0))):
        assert torch.equal(got, want.to(dt))
    # with an activation whose slope is 1 or 2: ds stays whole, and its sums exact
    y, saved = ops.linear(x, w, b, "lrelu", 2.0, save=True)
    s = X @ W.t() + b.double()
    assert torch.equal(y, torch.where(s > 0, s, 2 * s).to(dt))
    ds = D * torch.where(s > 0, 1.0, 2.0)
    for got, want in zip(ops.linear_backward(dy, x, w, saved, "lrelu", 2.0), (ds @ W, ds.t() @ X, ds.sum(0))):
        assert torch.equal(got, want.to(dt))


@pytest.mark.parametrize("dt", R.DTYPES)
def test_linear_large_forms(dt):
    run_linear(dt, 640, 704, 648, "none", res=False, bias=False, seed=1)
    run_linear(dt, 640, 704, 648, "lrelu", layout="strided", seed=2)
    run_linear(dt, 640, 700, 650, "none", layout="transposed", seed=3)
    full = run_linear(dt, 640, 704, 648, "xtanh", seed=4)
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, True, True)):
        part = run_linear(dt, 640, 704, 648, "xtanh", seed=4, need=need)
        assert all(b is None or torch.equal(a, b) for a, b in zip(full[-1], part[-1]))


def test_linear_large_rows_past_the_last_are_left_alone():
    """Results are written to (rows, out) exactly: what lies behind them in the same allocation keeps its values."""
    from ivae_amd import _lib
    m, k, n = 515, 1024, 513
    x, w = torch.randn(m, k, device=dev()), torch.randn(n, k, device=dev())
    for dt, code in ((F32, 0), (BF16, 1)):
        X, W = x.to(dt), w.to(dt)
        buf = torch.full((m * n + 4096,), 7.0, device=dev(), dtype=dt)
        lin, nb = ops._linear_plan(m, k, n, code, 0, .1, k, 0, 0, 0)
        ws = torch.empty(nb + 256, dtype=torch.uint8, device=dev())
        ws[nb:] = 7
        assert _lib.lib().ivae_linear(lin, X.data_ptr(), W.data_ptr(), None, None, buf.data_ptr(), None, ws.data_ptr(), nb,
                                      torch.cuda.current_stream().cuda_stream) == 0
        assert bool((buf[m * n:] == 7).all()) and bool((ws[nb:] == 7).all())
        R.close(buf[:m * n].view(m, n), R.linear64(X.cpu(), W.cpu(), None, "none", None)["y"], "y")


@pytest.mark.parametrize("dt", R.DTYPES)
@pytest.mark.parametrize("m,k,n", [(600, 1024, 520), (64, 8192, 520), (1200, 2048, 1100), (260, 16384, 640)])
def test_linear_large_keeps_nan_and_infinities(dt, m, k, n):
    g = torch.Generator().manual_seed(12)
    x, w, b, dy = normal(g, m, k, dtype=dt), normal(g, n, k, scale=.03, dtype=dt), normal(g, n, dtype=dt), normal(g, m, n, dtype=dt)
    want = R.linear64(x, w, b, "none", None, dy)
    x[1, 3], x[2, 0], w[4, 7], dy[5, 6] = float("nan"), float("inf"), float("inf"), -float("inf")
    y = ops.linear(on(x), on(w), on(b)).cpu()
    rows, cols = torch.tensor([i for i in range(m) if i not in (1, 2)]), torch.tensor([j for j in range(n) if j != 4])
    R.close(y[rows][:, cols], tuple(v[rows][:, cols] for v in want["y"]), "finite part")
    assert torch.isnan(y[1]).all()
    s = torch.where(w[:, 0].double() > 0, float("inf"), -float("inf"))
    assert torch.equal(y[2, cols].double(), s[cols])
    inf4 = torch.where(x[rows, 7].double() > 0, float("inf"), -float("inf"))
    assert torch.equal(y[rows, 4].double(), inf4)
    dx, dw, db = (t.cpu() for t in ops.linear_backward(on(dy), on(x), on(w)))
    rows2 = torch.tensor([i for i in range(m) if i != 5])
    ok = torch.tensor([j for j in range(k) if j != 7])                     # (column 7 meets the weight's infinity)
    R.close(dx[rows2][:, ok], tuple(v[rows2][:, ok] for v in want["dx"]), "dx")
    s = torch.where(w[6].double() > 0, -float("inf"), float("inf"))
    assert torch.equal(dx[5, ok].double(), s[ok])
    okw = torch.tensor([j for j in range(k) if j not in (0, 3)])
    rw = torch.tensor([j for j in range(n) if j != 6])
    R.close(dw[rw][:, okw], tuple(v[rw][:, okw] for v in want["dw"]), "dw")
    assert torch.isnan(dw[:, 3]).all() and not torch.isfinite(dw[6]).any()
    assert float(db[6]) == -float("inf")


@pytest.mark.parametrize("dt", R.DTYPES)
def test_linear_large_misaligned(dt):
    """Dense matrices that start off a 16-byte boundary, and rows at one whose first element is off it."""
    g = torch.Generator().manual_seed(14)
    m, k, n = 1024, 1024, 768
    mats = []
    for r, c in ((m, k), (n, k), (m, n)):
        t = torch.randint(-3, 4, (r, c), generator=g).to(dt)
        flat = torch.empty(r * c + 1, dtype=dt, device=dev())
        flat[1:].view(r, c).copy_(t.to(dev()))
        mats.append(flat[1:].view(r, c))
        wide = torch.zeros(r, c + 16, dtype=dt, device=dev())
        wide[:, 3:3 + c].copy_(t.to(dev()))
        mats.append(wide[:, 3:3 + c])
    for x, w, dy in (mats[0::2], mats[1::2]):
        X, W, D = x.double(), w.double(), dy.double()
        assert x.data_ptr() % 16 and torch.equal(ops.linear(x, w), (X @ W.t()).to(dt))
        for got, want in zip(ops.linear_backward(dy, x, w), (D @ W, D.t() @ X, D.sum(0))):
            assert torch.equal(got, want.to(dt))


@pytest.mark.parametrize("dt", R.DTYPES)
def test_linear_large_on_two_streams_and_in_graphs(dt):
    """Large calls at once on two streams, and two graphs captured from them and replayed together, give what one call alone gives."""
    g = torch.Generator().manual_seed(15)
    m, k, n = 1500, 1016, 1200
    sets = [tuple(normal(g, *s, scale=.2, dtype=dt).to(dev()) for s in ((m, k), (n, k), (m, n))) for _ in range(2)]

    def step(s):
        y, saved = ops.linear(s[0], s[1], None, "silu", residual=s[2], save=True)
        return y, *ops.linear_backward(s[2], s[0], s[1], saved, "silu")
    want = [[t.clone() for t in step(s)] for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        got = []
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(step(s))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))
        del got
    graphs, outs = [], []
    for s, st in zip(sets, streams):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            outs.append(step(s))
        graphs.append(gr)
    for _ in range(3):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(outs, want) for a, b in zip(x, y))
        step(sets[0])


def test_linear_fp32_range():
    """The three parts of a value keep its range: products near both ends of fp32's."""
    g = torch.Generator().manual_seed(13)
    x, w = normal(g, 512, 1024), normal(g, 512, 1024)
    for sx, sw in ((2.0 ** 100, 2.0 ** -100), (2.0 ** -60, 2.0 ** -40), (2.0 ** 60, 2.0 ** 50)):
        y = ops.linear(on(x * sx), on(w * sw))
        v, bound = R.linear64(x * sx, w * sw, None, "none", None)["y"]
        R.close(y, (v, bound), (sx, sw))


def test_linear_leading_dimensions_and_empty():
    g = torch.Generator().manual_seed(8)
    x, w, b = normal(g, 2, 3, 5, 24), normal(g, 10, 24), normal(g, 10)
    y, saved = ops.linear(x.to(dev()), w.to(dev()), b.to(dev()), "silu", save=True)
    assert y.shape == (2, 3, 5, 10) and saved.shape == y.shape
    R.close(y.reshape(-1, 10), R.linear64(x.reshape(-1, 24), w, b, "silu", None)["y"], "y")
    one = ops.linear(x[0, 0, 0].to(dev()), w.to(dev()), b.to(dev()), "silu")
    assert one.shape == (10,)
    R.close(one[None], R.linear64(x[0, 0, :1], w, b, "silu", None)["y"], "y")
    e = torch.empty(0, 24, device=dev())
    y, saved = ops.linear(e, w.to(dev()), b.to(dev()), "silu", save=True)
    assert y.shape == (0, 10)
    dx, dw, db = ops.linear_backward(torch.empty(0, 10, device=dev()), e, w.to(dev()), saved, "silu")
    assert dx.shape == (0, 24) and float(dw.abs().sum()) == 0 and float(db.abs().sum()) == 0 and dw.shape == w.shape
    # one row repeated (stride 0), and the expanded gradient that a sum() hands back
    xr = x[0, 0, :1].to(dev()).expand(7, 24)
    dy = torch.ones(1, 1, device=dev()).expand(7, 10)
    want = R.linear64(xr.cpu().contiguous(), w, b, "none", None, dy.cpu().contiguous())
    R.close(ops.linear(xr, w.to(dev()), b.to(dev())), want["y"], "y")
    for name, t in zip(("dx", "dw", "db"), ops.linear_backward(dy, xr, w.to(dev()))):
        R.close(t, want[name], name)


@pytest.mark.parametrize("dt", R.DTYPES)
@pytest.mark.parametrize("m,k,n", [(5, 40, 30), (200, 256, 320)])
def test_linear_keeps_nan_and_infinities_where_they_belong(dt, m, k, n):
    """A row with a NaN, a row with an infinity, a weight row with an infinity: the others are what they are without them."""
    g = torch.Generator().manual_seed(9)
    x, w, b = normal(g, m, k, dtype=dt), normal(g, n, k, scale=.1, dtype=dt), normal(g, n, dtype=dt)
    clean = ops.linear(on(x), on(w), on(b), "lrelu").cpu()
    x2, w2 = x.clone(), w.clone()
    x2[1, 3] = float("nan")
    x2[2, 0] = float("inf")
    w2[4, 7] = float("inf")
    y = ops.linear(on(x2), on(w2), on(b), "lrelu").cpu()
    rows, cols = [i for i in range(m) if i not in (1, 2)], [j for j in range(n) if j != 4]
    assert torch.equal(y[rows][:, cols], clean[rows][:, cols])
    assert torch.isnan(y[1]).all()
    s = torch.where(w[:, 0].double() > 0, float("inf"), -float("inf"))
    assert torch.equal(y[2, cols].double(), s[cols]) and not torch.isfinite(y[rows][:, 4]).any()


@pytest.mark.parametrize("dt", [BF16, F16])
def test_linear_saved_clamps_and_keeps_the_side(dt):
    """Pre-activations beyond fp16's range and far below it: the slope of lrelu is that of their side, gelu's is 0 or 1."""
    s = torch.tensor([6e4, -6e4, 1e-7, -1e-7, 0.0], dtype=dt)[:, None]
    x, w = s.to(dev()), torch.full((1, 1), 3.0, dtype=dt, device=dev())
    dy = torch.ones(5, 1, dtype=dt, device=dev())
    for act, want in (("lrelu", [1, .1, 1, .1, .1]), ("gelu", [1, 0, .5, .5, .5])):
        y, saved = ops.linear(x, w, None, act, save=True)
        assert torch.isfinite(saved).all()
        dx, _, _ = ops.linear_backward(dy, x, w, saved, act)
        # ds and dx are rounded once each: 2 u; 3 * ds is the product
        assert torch.allclose(dx.float().cpu().view(-1), 3 * torch.tensor(want), rtol=2.5 * R.u(dt), atol=1e-5), (act, dx)


def test_linear_is_deterministic_and_streams_agree():
    args = run_linear(BF16, 700, 300, 200, "gelu", seed=11)
    X, W, B, Rr, D, saved, y, grads = args
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y2 = ops.linear(X, W, B, "gelu", R.SLOPE, residual=Rr)
        g2 = ops.linear_backward(D, X, W, saved, "gelu")
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, y2) and all(torch.equal(a, b) for a, b in zip(grads, g2))


def test_linear_refuses_what_it_does_not_serve():
    x, w = torch.zeros(4, 6, device=dev()), torch.zeros(5, 6, device=dev())
    y, saved = ops.linear(x, w, None, "gelu", save=True)
    for call, err in ((lambda: ops.linear(x, w.t()), ValueError), (lambda: ops.linear(x, w, torch.zeros(6, device=dev())), ValueError),
                      (lambda: ops.linear(x, w, residual=torch.zeros(5, device=dev())), ValueError), (lambda: ops.linear(x, w, activation="relu"), ValueError),
                      (lambda: ops.linear(x, w.half()), TypeError), (lambda: ops.linear(x, w, torch.zeros(5)), RuntimeError),
                      (lambda: ops.linear(x, w, torch.zeros(5, device=dev(), dtype=BF16)), TypeError),
                      (lambda: ops.linear(torch.zeros(4, 0, device=dev()), torch.zeros(5, 0, device=dev())), ValueError),
                      (lambda: ops.linear_backward(y, x, w, None, "gelu"), ValueError), (lambda: ops.linear_backward(y[:3], x, w), ValueError),
                      (lambda: ops.linear_backward(y, x, w, saved.half(), "gelu"), TypeError)):
        with pytest.raises(err):
            call()


# ---- layer norm ---------------------------------------------------------------------------------------------------------


def run_norm(dt, m, d, wdtype=None, affine=True, layout="dense", seed=0, shift=.5, eps=1e-5, residual=False):
    g = torch.Generator().manual_seed(seed)
    wt = wdtype or dt
    x = normal(g, m, d, scale=1.5, dtype=dt) + torch.tensor(shift, dtype=dt)
    w = (1 + normal(g, d, scale=.2)).to(wt) if affine else None
    b = normal(g, d, scale=.2, dtype=wt) if affine else None
    dy = normal(g, m, d, dtype=dt)
    r = normal(g, m, d, dtype=dt) if residual else None
    want = R.norm64(x, w, b, eps, dy, r, wt if affine else None)
    X, D, Rr = on(x, layout), on(dy, layout), on(r, layout)
    y, stats = ops.layer_norm(X, on(w), on(b), eps, save=True)
    R.close(y, want["y"], "y")
    assert torch.equal(y, ops.layer_norm(X, on(w), on(b), eps))
    got = ops.layer_norm_backward(D, X, stats, on(w), residual=Rr)
    for name, t in zip(("dx", "dw", "db"), got):
        R.close(t, want[name], name)
    again = ops.layer_norm_backward(D, X, stats, on(w), residual=Rr)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    return X, D, stats, got


@pytest.mark.parametrize("m,d", [(1, 1), (1, 2), (5, 1), (64, 50), (3, 255), (70, 256), (37, 257), (130, 1000), (9, 1024), (33, 1025), (3, 4096), (5, 4099),
                                 (3, 5000), (2, 16384), (700, 200), (3000, 24), (1, 20001), (6, 20001),
                                 (3, 5001), (600, 4090), (40, 16381), (10500, 200), (2200, 1000), (1100, 2000), (520, 4096)])
@pytest.mark.parametrize("dt", R.DTYPES)
def test_layer_norm_sizes(dt, m, d):
    run_norm(dt, m, d, seed=m + d)


@pytest.mark.parametrize("dt", R.DTYPES)
def test_layer_norm_forms(dt):
    run_norm(dt, 40, 100, affine=False, seed=1)
    run_norm(dt, 40, 300, wdtype=F32, seed=2, residual=True)
    run_norm(dt, 33, 129, layout="strided", seed=3, residual=True)
    run_norm(dt, 33, 128, layout="transposed", seed=4)
    run_norm(dt, 5, 20001, wdtype=F32, seed=6, residual=True)
    run_norm(dt, 33, 128, seed=5, eps=0.5)


def test_layer_norm_constant_rows_and_parts():
    x = torch.full((4, 33), 3.25, device=dev())
    y, stats = ops.layer_norm(x, save=True)
    assert float(y.abs().max()) == 0 and torch.equal(stats[0].cpu(), torch.full((4,), 3.25))
    assert torch.allclose(stats[1].cpu(), torch.full((4,), 1e5 ** .5), rtol=1e-6)
    X, D, stats, full = run_norm(F32, 50, 70, seed=6, affine=False)
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, False, False)):
        part = ops.layer_norm_backward(D, X, stats, need=need)
        assert all((b is None) if not n else torch.equal(a, b) for a, b, n in zip(full, part, need))
    e = torch.empty(0, 9, device=dev())
    y, stats = ops.layer_norm(e, save=True)
    dx, dw, db = ops.layer_norm_backward(e, e, stats)
    assert y.shape == dx.shape == (0, 9) and float(dw.abs().sum()) == 0 and float(db.abs().sum()) == 0


@pytest.mark.parametrize("dt", R.DTYPES)
@pytest.mark.parametrize("m,d", [(1, 8), (24, 64), (25, 64), (23, 50), (6, 2048), (3, 1037), (2, 16384), (3, 16381)])
def test_layer_norm_few_rows(dt, m, d):
    """Up to six rows of a block's share of threads are one block's, which writes the weight's gradients itself."""
    for wdtype in (dt, F32):
        X, D, stats, full = run_norm(dt, m, d, wdtype=wdtype, seed=m + d, residual=True)
        w = torch.ones(d, device=dev(), dtype=wdtype)
        one = ops.layer_norm_backward(D, X, stats, w)
        for need in ((True, False, False), (False, True, False), (False, False, True), (False, False, False)):
            part = ops.layer_norm_backward(D, X, stats, w, need=need)
            assert all((b is None) if not n else torch.equal(a, b) for a, b, n in zip(one, part, need))
        assert all(torch.equal(a, b) for a, b in zip(one[1:], full[1:]))          # (they do not depend on the weight)


def test_layer_norm_nan_stays_in_its_row():
    g = torch.Generator().manual_seed(7)
    x = normal(g, 20, 300).to(dev())
    clean = ops.layer_norm(x)
    x[3, 5], x[9, 299] = float("nan"), float("inf")
    y = ops.layer_norm(x)
    rows = [i for i in range(20) if i not in (3, 9)]
    assert torch.equal(y[rows], clean[rows]) and torch.isnan(y[3]).all() and torch.isnan(y[9]).any()


def test_layer_norm_refuses_what_it_does_not_serve():
    x, w = torch.zeros(4, 6, device=dev(), dtype=BF16), torch.ones(6, device=dev())
    _, stats = ops.layer_norm(x, w, save=True)
    for call, err in ((lambda: ops.layer_norm(x, w.half()), TypeError), (lambda: ops.layer_norm(x, w, w.to(BF16)), TypeError),
                      (lambda: ops.layer_norm(x, w[:5]), ValueError), (lambda: ops.layer_norm(x[:, :0]), ValueError),
                      (lambda: ops.layer_norm(x, w.cpu()), RuntimeError), (lambda: ops.layer_norm_backward(x, x[:3], stats), ValueError),
                      (lambda: ops.layer_norm_backward(x, x, stats[:1]), ValueError), (lambda: ops.layer_norm_backward(x.float(), x, stats), TypeError)):
        with pytest.raises(err):
            call()


@pytest.mark.parametrize("dt", R.DTYPES)
@pytest.mark.parametrize("d", [1031, 2048])
def test_results_beyond_the_cache(dt, d):
    """Results of 96 MB and more are stored another way; their rows, and their elements, are those of the two halves."""
    m = 2 * (((100 << 20) // (d * torch.finfo(dt).bits // 8) + 1) // 2)
    g = torch.Generator(device=dev()).manual_seed(d)
    x, dy, r = (torch.randn(m, d, device=dev(), generator=g).to(dt) for _ in range(3))
    w = torch.randn(d, device=dev(), generator=g).to(dt)
    parts = slice(0, m // 2), slice(m // 2, m)
    y, stats = ops.layer_norm(x, w, w, save=True)
    dx = ops.layer_norm_backward(dy, x, stats, w, residual=r)[0]
    z = ops.dropout(x, .25, 7, 1, residual=r)
    keep = ops.dropout(torch.ones_like(x), .25, 7, 1) != 0
    assert abs(float(keep.float().mean()) - .75) < 1e-3
    for i, p in enumerate(parts):
        yp, sp = ops.layer_norm(x[p], w, w, save=True)
        assert torch.equal(y[p], yp) and torch.equal(stats[:, p], sp)
        assert torch.equal(dx[p], ops.layer_norm_backward(dy[p], x[p], sp, w, residual=r[p])[0])
    n = m // 2 * d
    assert torch.equal(z.view(-1)[:n], ops.dropout(x.view(-1)[:n], .25, 7, 1, residual=r.view(-1)[:n]))
    v = torch.where(keep, x.float() * (4 / 3), 0.) + r.float()
    # 4 / 3, the product and the sum are rounded to 24 bits on each side, the result to its type
    bound = R.u(dt) * v.abs() + R.tiny(dt) + 8 * R.U32 * (v.abs() + r.float().abs())
    assert bool(((z.float() - v).abs() <= bound).all())


# ---- dropout ------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("n", [1, 3, 4, 7, 8, 9, 64, 1001, 12800, 70001])
@pytest.mark.parametrize("dt", R.DTYPES)
def test_dropout_mask_and_values(dt, n):
    g = torch.Generator().manual_seed(n)
    x, r = normal(g, n, dtype=dt), normal(g, n, dtype=dt)
    for p, seed, offset in ((.1, 0, 0), (.5, 2 ** 64 - 3, 2 ** 40 + 5), (.937, -7, -1), (0., 1, 1), (1., 1, 1), (2.0 ** -32, 5, 5)):
        k = R.keep(n, p, seed, offset)
        scaled = x.double() / (1 - p) if p < 1 else torch.zeros(n, dtype=torch.float64)
        value = torch.where(k, scaled, torch.zeros_like(scaled))
        # 1 / (1 - p) is rounded to fp32, the product (and the sum) once more, then to the type
        bound = R.u(dt) * value.abs() + R.tiny(dt) + 3 * R.U32 * value.abs()
        y = ops.dropout(on(x), p, seed, offset)
        assert torch.equal((y == 0).cpu() | (x == 0), ~k | (x == 0))
        R.close(y, (value, bound), "y")
        assert torch.equal(y, ops.dropout_backward(on(x), p, seed, offset))
        v2 = value + r.double()
        R.close(ops.dropout(on(x), p, seed, offset, residual=on(r)), (v2, R.u(dt) * v2.abs() + R.tiny(dt) + 3 * R.U32 * (value.abs() + r.double().abs())), "y + residual")


def test_dropout_drops_nan_and_does_not_depend_on_shape():
    x = torch.full((40, 50), float("nan"), device=dev())
    y = ops.dropout(x, .3, 9, 4)
    k = R.keep(2000, .3, 9, 4).view(40, 50)
    assert torch.equal(torch.isnan(y).cpu(), k) and float(y[~k.to(dev())].abs().sum()) == 0
    x = torch.randn(40, 50, device=dev())
    a = ops.dropout(x, .3, 9, 4)
    assert torch.equal(a, ops.dropout(x.view(-1), .3, 9, 4).view(40, 50))
    assert torch.equal(a, ops.dropout(x.t().contiguous().t(), .3, 9, 4))
    assert not torch.equal(a, ops.dropout(x, .3, 9, 5)) and not torch.equal(a, ops.dropout(x, .3, 10, 4))
    assert ops.dropout(x[:0], .3, 9, 4).shape == (0, 50)


def test_dropout_offset_in_device_memory():
    x = torch.randn(3000, device=dev())
    off = torch.tensor([2 ** 33 + 7], device=dev())
    assert torch.equal(ops.dropout(x, .4, 3, off), ops.dropout(x, .4, 3, 2 ** 33 + 7))
    for bad, err in ((off.int(), TypeError), (torch.zeros(2, dtype=torch.int64, device=dev()), ValueError), (torch.zeros(1, dtype=torch.int64), RuntimeError)):
        with pytest.raises(err):
            ops.dropout(x, .4, 3, bad)
    for p in (-.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            ops.dropout(x, p, 3)
    with pytest.raises(ValueError):
        ops.dropout(x, .1, 3, residual=x[:5])


def test_dropout_rate():
    """The kept share of 4 million draws: a binomial's 5 sigma around 1 - p."""
    n = 1 << 22
    y = ops.dropout(torch.ones(n, device=dev()), .3, 12345, 678)
    assert abs(float((y > 0).double().mean()) - .7) < 5 * (.21 / n) ** .5


# ---- together -----------------------------------------------------------------------------------------------------------


def test_block_replays_from_a_graph():
    """The three operators, forward and backward, captured once: every replay equals the eager run on the same inputs, with eager work
    between the replays, and the dropout mask advances with the offset in device memory."""
    g = torch.Generator().manual_seed(21)
    m, d, h = 96, 80, 160
    x, dy = normal(g, m, d).to(dev()), normal(g, m, d).to(dev())
    gam, bet, w1, b1, w2, b2 = (normal(g, *s, scale=.3).to(dev()) for s in ((d,), (d,), (h, d), (h,), (d, h), (d,)))
    off = torch.zeros(1, dtype=torch.int64, device=dev())

    def step():
        t, st = ops.layer_norm(x, gam, bet, save=True)
        a, pre = ops.linear(t, w1, b1, "gelu", save=True)
        y = ops.dropout(ops.linear(a, w2, b2), .2, 77, off, residual=x)
        do = ops.dropout_backward(dy, .2, 77, off)
        da, dw2, db2 = ops.linear_backward(do, a, w2)
        dn, dw1, db1 = ops.linear_backward(da, t, w1, pre, "gelu")
        dx, dg, dc = ops.layer_norm_backward(dn, x, st, gam, residual=dy)
        return y, dx, dg, dc, dw1, db1, dw2, db2
    step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            out = step()
        with torch.cuda.graph(second, stream=side):
            out2 = step()
    seen = []
    for i in range(4):
        x.add_(.25 * i)
        off.fill_(10 + i)
        graph.replay()
        second.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) and torch.equal(c, b) for a, b, c in zip(out, want, out2)), i
        seen.append(out[0].clone())
    assert not torch.equal(seen[0], seen[1])


def _mlp64(m, x, masks=None):
    """The MLP's formula in 64 bits, with autograd."""
    h = x
    for c, fc in enumerate(m.fc):
        w, b = fc.weight.detach().cpu().double().requires_grad_(), fc.bias.detach().cpu().double().requires_grad_()
        m.ref.append((fc.weight, w)), m.ref.append((fc.bias, b))
        t = h
        if m.norm is not None and c:
            nw, nb = (p.detach().cpu().double().requires_grad_() for p in (m.norm[c - 1].weight, m.norm[c - 1].bias))
            m.ref.append((m.norm[c - 1].weight, nw)), m.ref.append((m.norm[c - 1].bias, nb))
            t = torch.nn.functional.layer_norm(t, (t.shape[-1],), nw, nb, m.norm[c - 1].eps)
        t = t @ w.t() + b
        if c == m.n_layers - 1:
            return t
        t = R.act64(t, m.activation[c], m.slope)[0]
        if masks is not None:
            t = torch.where(masks[c].view(t.shape), t / (1 - m.dropout), torch.zeros_like(t))
        h = t + h if m.residual and fc.in_features == fc.out_features else t


@pytest.mark.parametrize("act", ["xtanh", "gelu"])
@pytest.mark.parametrize("opts", [dict(layer_norm=True), dict(residual=True), dict(layer_norm=True, residual=True, dropout=.25)])
def test_mlp_operators_forward_and_gradients(act, opts):
    torch.manual_seed(5)
    m = MLP(12, 5, 40, 4, activation=act, **opts).to(dev())
    x = torch.randn(64, 12)
    X = x.to(dev()).requires_grad_()
    masks = None
    if m.dropout:
        torch.manual_seed(99)
        seed = int(torch.randint(2 ** 63 - 1, ()))
        masks = [R.keep(64 * 40, m.dropout, seed, c) for c in range(3)]
        torch.manual_seed(99)
    y = m(X)
    y.square().sum().backward()
    m.ref = []
    x64 = x.double().requires_grad_()
    y64 = _mlp64(m, x64, masks)
    y64.square().sum().backward()
    # four layers of sums over at most 64 rows or 40 columns, each off by at most 80 roundings of its magnitudes, and gradients through
    # as many again: 8 * 80 * 2^-24 = 4e-5 of the largest magnitude
    tol = lambda v: 4e-5 * float(v.abs().max())  # noqa: E731
    assert float((y.detach().cpu().double() - y64.detach()).abs().max()) < tol(y64.detach())
    assert float((X.grad.cpu().double() - x64.grad).abs().max()) < tol(x64.grad)
    for p, q in m.ref:
        assert float((p.grad.cpu().double() - q.grad).abs().max()) < tol(q.grad), p.shape
    m.eval()
    assert torch.equal(m(X), m(X)) and (m.dropout == 0 or not torch.equal(m(X), y))


def test_mlp_operators_differences():
    """Directional central differences of the kernels' own forward pass against their gradients: at h = 2^-6 the truncation is
    h^2 / 6 times a third derivative of order 10 (4e-4), the rounding of the two sums 2^-24 sqrt(320) 20 / h = 1e-3, relative to
    a directional derivative of order 10: 1e-3 with a margin of 5."""
    torch.manual_seed(6)
    m = MLP(10, 5, 32, 3, activation="xtanh", layer_norm=True, residual=True).to(dev())
    x, dy = torch.randn(64, 10, device=dev()), torch.randn(64, 5, device=dev())
    X = x.clone().requires_grad_()
    (m(X) * dy).sum().backward()
    v = torch.randn_like(x)
    v /= v.norm()
    h = 2.0 ** -6
    with torch.no_grad():
        up, dn = ((m(x + s * h * v).double() * dy.double()).sum() for s in (1, -1))
    got, want = float((up - dn) / (2 * h)), float((X.grad.double() * v.double()).sum())
    assert abs(got - want) < 5e-3 * max(1.0, float(X.grad.norm())), (got, want)


def test_mlp_operators_bf16_and_frozen_parts():
    torch.manual_seed(7)
    m = MLP(16, 8, 32, 3, activation="silu", layer_norm=True, residual=True).to(dev()).to(BF16)
    x = torch.randn(20, 16, device=dev(), dtype=BF16)
    m.fc[1].weight.requires_grad_(False)
    y = m(x)
    assert y.dtype == BF16
    y.float().sum().backward()
    assert m.fc[1].weight.grad is None and all(p.grad is not None and p.grad.dtype == BF16 for n, p in m.named_parameters() if n != "fc.1.weight")
    with torch.no_grad():
        assert torch.equal(m(x), y)
    g = torch.autograd.grad(m(x.requires_grad_()).float().sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError):                   # no second derivatives
        g.float().sum().backward()


def test_mlp_operators_under_capture():
    """The forward pass of eval() captures; autograd and dropout say what to do instead."""
    torch.manual_seed(8)
    m = MLP(16, 8, 32, 3, activation="silu", layer_norm=True, residual=True, dropout=.5).to(dev()).eval()
    x = torch.randn(20, 16, device=dev())
    with torch.no_grad():
        want = m(x)
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            with torch.no_grad():
                out = m(x)
            with pytest.raises(RuntimeError, match="capture"):
                m(x)
            with pytest.raises(RuntimeError, match="mask"), torch.no_grad():
                m.train()(x)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
