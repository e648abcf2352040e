"""How exact the tensor operators are where worst-case bounds of long sums see nothing: root mean squares of errors against the rounding
of the results alone, values at the ends of a type's range, infinities that meet a zero of a split value."""
import pytest
import torch

from ivae_amd import ops
from tests import operator_ref as R

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
# (rows, in, out) that the 64 x 64 kernels take, and such that the large kernels' backward passes take
SIZES = [(96, 120, 104), (300, 33, 77), (1024, 768, 520), (1003, 777, 531)]
GRADS = ("dx", "dw", "db")


def dev():
    return torch.device("cuda:0")


def normal(g, *shape, scale=1.0, dtype=F32):
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def step(v, dtype):
    """Distance of the type's numbers around v (64 bits)."""
    f = torch.finfo(dtype)
    e = torch.floor(torch.log2(v.abs().clamp(min=f.smallest_normal)))
    return torch.exp2(e) * f.eps


def only_rounded(got, want, dtype, what, noise=0.0):
    """A result that is rounded once is off by a uniform draw of half a step: step / sqrt 12 in the root mean square.  10 % are left for the
    sums in 32 bits and for the draw (1e5 of them vary by 0.3 %); a second rounding of equal size would make it 41 %.  noise: what the sums add."""
    got = got.detach().cpu().double()
    assert torch.isfinite(got).all(), what
    rms = (got - want).square().mean().sqrt()
    alone = (step(want, dtype).square().mean() / 12).sqrt()
    # few results (db): the draw's own spread, 5 sigma of a mean of n squares (their variance is 0.8 of the mean squared)
    few = 5 * (0.8 / want.numel()) ** 0.5
    bound = ((1.1 + few) * alone.square() + noise ** 2).sqrt() * 1.05
    assert rms <= bound, (what, float(rms / alone))


def formula(x, w, b, act, dy, slope=R.SLOPE):
    X, W, D = x.double(), w.double(), dy.double()
    s = X @ W.t() + (b.double() if b is not None else 0.0)
    a, k = R.act64(s, act, slope)
    ds = D * k
    return {"y": a, "dx": ds @ W, "dw": ds.t() @ X, "db": ds.sum(0), "s": s}


def gradients(x, w, b, act, dy, slope=R.SLOPE):
    X, W, D = x.to(dev()), w.to(dev()), dy.to(dev())
    _, saved = ops.linear(X, W, b.to(dev()) if b is not None else None, act, slope, save=True)
    return dict(zip(GRADS, ops.linear_backward(D, X, W, saved, act, slope))), saved


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("act", R.ACTS)
@pytest.mark.parametrize("dt", [BF16, F16])
def test_gradients_are_rounded_once(dt, act, m, k, n):
    g = torch.Generator().manual_seed(m + n)
    x, w, b, dy = normal(g, m, k, dtype=dt), normal(g, n, k, scale=k ** -0.5, dtype=dt), normal(g, n, scale=.3, dtype=dt), normal(g, m, n, dtype=dt)
    if act == "lrelu":          # no pre-activation near the kink, where the order of a sum decides the side
        b = torch.where(b >= 0, 1.0, -1.0).to(dt) * 8
    want, (got, _) = formula(x, w, b, act, dy), gradients(x, w, b, act, dy)
    for name in GRADS:
        only_rounded(got[name], want[name], dt, (name, act))


@pytest.mark.parametrize("dt", R.DTYPES)
def test_saved_holds_32_bits(dt):
    """The pre-activation that the backward pass takes act' of, in the tail of gelu's slope: there s off by 2^-9 (half a step of fp16) moves act' by
    |s| 2^-9, twice the rounding of a bf16 result.  Each gradient here is one product; the evaluation of act' is off by at most 2^-10 of it."""
    x = torch.linspace(-4.25, -4.03125, 512).to(dt)[:, None]
    w, b, dy = torch.ones(1, 1, dtype=dt), torch.full((1,), 2.0 ** -9).to(dt), torch.ones(512, 1, dtype=dt)
    want = formula(x, w, b, "gelu", dy)
    got, saved = gradients(x, w, b, "gelu", dy)
    assert saved.dtype == F32 and bool(((saved.cpu().double() - want["s"]).abs() <= R.U32 * 4.25).all())
    err = (got["dx"].cpu().double() - want["dx"]).abs()
    assert bool((err <= (R.u(dt) + 2.0 ** -10) * want["dx"].abs() + R.tiny(dt)).all()), float((err / want["dx"].abs()).max())


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("scale", [2.0 ** -17, 2.0 ** -20])
def test_small_fp16_gradients_keep_their_digits(scale, m, k, n):
    """dy among fp16's subnormal numbers, and products that the type holds: act'(s) dy has 32 bits on its way into them."""
    g = torch.Generator().manual_seed(5)
    x, w = normal(g, m, k, scale=2.0 ** 6, dtype=F16), normal(g, n, k, scale=2.0 ** 8, dtype=F16)
    dy = normal(g, m, n, scale=scale, dtype=F16)
    b = normal(g, n, scale=.3, dtype=F16)
    x[:, 1:] = 0                                # (so that s stays moderate: one product of 2^-8 and 2^8)
    x[:, 0] = normal(g, m, scale=2.0 ** -8, dtype=F16)
    want, (got, _) = formula(x, w, b, "gelu", dy), gradients(x, w, b, "gelu", dy)
    assert float(want["dx"].abs().mean()) > 2.0 ** -13
    only_rounded(got["dx"], want["dx"], F16, "dx")
    x = normal(g, m, k, scale=2.0 ** 12, dtype=F16)
    w = normal(g, n, k, scale=2.0 ** -12 * k ** -0.5, dtype=F16)
    want, (got, _) = formula(x, w, b, "gelu", dy), gradients(x, w, b, "gelu", dy)
    # (s is a sum in 32 bits: relative 2^-24 sqrt(k) of numbers of order 1)
    only_rounded(got["dw"], want["dw"], F16, "dw")


@pytest.mark.parametrize("m,k,n", SIZES)
def test_smallest_bf16_gradients_keep_their_digits(m, k, n):
    """dy at the end of bf16's range, where a second number at the first one's scale would have no bits left, and products far inside of it."""
    g = torch.Generator().manual_seed(5)
    x, w = normal(g, m, k, dtype=BF16), normal(g, n, k, scale=k ** -0.5, dtype=BF16)
    dy = normal(g, m, n, dtype=F32).mul(2.0 ** -125).to(BF16)
    big = torch.ldexp(x.float(), torch.tensor(60)).to(BF16)
    _, saved = ops.linear(x.to(dev()), w.to(dev()), None, "gelu", save=True)
    want = formula(x, w, None, "gelu", dy)["dw"] * 2.0 ** 60
    _, got, _ = ops.linear_backward(dy.to(dev()), big.to(dev()), w.to(dev()), saved, "gelu")
    only_rounded(got * 2.0 ** 60, want * 2.0 ** 60, BF16, "dw")


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("act,slope", [("gelu", .1), ("lrelu", 2.0), ("lrelu", 1000.0), ("xtanh", 30.0), ("silu", .1)])
def test_large_fp16_gradients_stay_finite(act, slope, m, k, n):
    """act'(s) dy beyond 65504, in products that the type holds."""
    g = torch.Generator().manual_seed(6)
    x, w = normal(g, m, k, scale=2.0 ** -9, dtype=F16), normal(g, n, k, scale=2.0 ** -8, dtype=F16)
    b = torch.full((n,), 1.4 if act != "lrelu" else -1.4, dtype=F16)
    dy = (torch.where(torch.rand(m, n, generator=g) < .5, 1.0, -1.0) * 60000 * (1 - torch.rand(m, n, generator=g) / 16)).to(F16)
    if slope > 2:
        dy = (dy.float() / slope * 2).to(F16)
    want, (got, _) = formula(x, w, b, act, dy, slope), gradients(x, w, b, act, dy, slope)
    for name in ("dx", "dw"):
        assert float(want[name].abs().max()) < 65000
        only_rounded(got[name], want[name], F16, (name, act))


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("dt", R.DTYPES)
def test_infinities_in_gradients_with_an_activation(dt, m, k, n):
    """x or w infinite where act'(s) dy is a number that the type holds: each product is that infinity, not 0 times it."""
    g = torch.Generator().manual_seed(7)
    x, w, dy = normal(g, m, k, dtype=dt), normal(g, n, k, scale=.03, dtype=dt), normal(g, m, n, dtype=dt)
    dy[dy == 0] = 1
    b = normal(g, n, dtype=dt)
    X, W, D = x.to(dev()), w.to(dev()), dy.to(dev())
    _, saved = ops.linear(X, W, b.to(dev()), "lrelu", 0.5, save=True)
    clean = ops.linear_backward(D, X, W, saved, "lrelu", 0.5)
    ds = dy.double() * torch.where(saved.cpu() > 0, 1.0, 0.5)        # half a value is a value of the type
    X[3, 5], W[7, 2] = float("inf"), -float("inf")
    dx, dw, db = ops.linear_backward(D, X, W, saved, "lrelu", 0.5)
    assert torch.equal(dw[:, 5].cpu().double(), torch.sign(ds[3]) * float("inf"))
    assert torch.equal(dx[:, 2].cpu().double(), -torch.sign(ds[:, 7]) * float("inf"))
    cols, ok = [j for j in range(k) if j != 5], [j for j in range(k) if j != 2]
    want = {"dx": ds @ w.double(), "dw": ds.t() @ x.double()}
    for name, t, keep in (("dx", dx, ok), ("dw", dw, cols)):
        if dt == F32:
            mag = ds.abs() @ w.double().abs() if name == "dx" else ds.abs().t() @ x.double().abs()
            R.close(t[:, keep], (want[name][:, keep], (R.U32 * ((m if name == "dw" else n) + 16) * mag)[:, keep]), name)
        else:
            only_rounded(t[:, keep], want[name][:, keep], dt, name)
    assert torch.equal(db, clean[2])
    # ... and an infinite gradient
    D[4, 6] = float("inf")
    X[3, 5], W[7, 2] = x[3, 5], w[7, 2]
    dx, dw, db = ops.linear_backward(D, X, W, saved, "lrelu", 0.5)
    assert torch.equal(dx[4].cpu().double(), torch.sign(w[6].double()) * float("inf"))
    assert torch.equal(dw[6].cpu().double(), torch.sign(x[4].double()) * float("inf")) and float(db[6]) == float("inf")
    assert torch.isfinite(dx[:4]).all() and torch.isfinite(dx[5:]).all() and torch.isfinite(dw[:6]).all() and torch.isfinite(dw[7:]).all()


@pytest.mark.parametrize("m,k,n", SIZES + [(64, 50, 50), (6000, 17, 19)])
@pytest.mark.parametrize("act", ["none", "gelu"])
@pytest.mark.parametrize("dt", R.DTYPES)
def test_gradients_without_the_operands_that_they_do_not_need(dt, act, m, k, n):
    """The bias gradient needs neither x nor w, dx no x, dw no w: the C entry takes NULL for them, and the gradients are the same."""
    from ivae_amd import _lib
    g = torch.Generator().manual_seed(8)
    X, W, D = (t.to(dev()) for t in (normal(g, m, k, dtype=dt), normal(g, n, k, scale=k ** -0.5, dtype=dt), normal(g, m, n, dtype=dt)))
    _, saved = ops.linear(X, W, None, act, save=True)
    want = ops.linear_backward(D, X, W, saved, act)
    lin, nb = ops._linear_plan(m, k, n, ops.DTYPE_IDS[dt], _lib.LINEAR_ACT_IDS[act], R.SLOPE, k, 0, n, 1)
    ws = torch.empty(max(nb, 16), dtype=torch.uint8, device=dev())
    for need in ((False, False, True), (True, False, True), (False, True, True), (True, False, False), (False, True, False)):
        out = [torch.full_like(t, 7.0) if w else None for t, w in zip(want, need)]
        rc = _lib.lib().ivae_linear_backward(lin, D.data_ptr(), X.data_ptr() if need[1] else None, W.data_ptr() if need[0] else None,
                                             saved.data_ptr() if saved is not None else None, *[t.data_ptr() if t is not None else None for t in out],
                                             ws.data_ptr(), nb, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        for name, a, b in zip(GRADS, want, out):
            assert b is None or torch.equal(a, b), (name, need)


# products that the 64 x 64 kernel takes, and such that the split kernels take (forward pass: 5e9 operations and more, odd sizes 2e9)
@pytest.mark.parametrize("m,k,n", [(96, 120, 104), (1024, 2048, 1300), (1100, 1501, 1003)])
@pytest.mark.parametrize("ex,ew", [(0, 0), (-60, -50), (-112, 100), (-118, 100), (-121, 100), (100, -125), (-130, 110), (-118, 0), (0, -122)])
def test_fp32_keeps_its_digits_down_to_the_smallest_numbers(m, k, n, ex, ew):
    """x 2^ex and w 2^ew of unit values, the gradient at x's scale: a sum of n products of 24-bit numbers is off by a walk of sqrt(n) half steps
    or less.  Numbers below 2^-126 have fewer bits themselves; the formula takes them as they are.  db and results below 2^-126 are left out."""
    g = torch.Generator().manual_seed(m)
    x, w, dy = (torch.ldexp(normal(g, *s), torch.tensor(e)) for s, e in (((m, k), ex), ((n, k), ew), ((m, n), ex)))
    got = {"y": ops.linear(x.to(dev()), w.to(dev()))}
    got["dx"], got["dw"], _ = ops.linear_backward(dy.to(dev()), x.to(dev()), w.to(dev()))
    up = lambda t, e: torch.ldexp(t.double(), torch.tensor(-e))  # noqa: E731
    X, W, D = up(x, ex), up(w, ew), up(dy, ex)
    for name, want, e, terms in (("y", X @ W.t(), ex + ew, k), ("dx", D @ W, ex + ew, n), ("dw", D.t() @ X, 2 * ex, m)):
        if -120 < e < 110:
            rms = float((up(got[name].cpu(), e) - want).square().mean().sqrt() / want.square().mean().sqrt())
            assert rms <= R.U32 * terms ** 0.5, (name, rms)


def test_fp32_tiny_rows_among_ordinary_ones():
    """Rows whose values have bits that a bf16 number cannot hold, among rows of unit scale and rows of zeros: each is right by itself."""
    g = torch.Generator().manual_seed(9)
    m, k, n = 1100, 1501, 1003
    x, w = normal(g, m, k), torch.ldexp(normal(g, n, k), torch.tensor(20))
    x[300:310] = torch.ldexp(x[300:310], torch.tensor(-120))
    x[700:800] = 0
    w[5] = torch.ldexp(w[5], torch.tensor(-140))
    y = ops.linear(x.to(dev()), w.to(dev())).cpu().double()
    want, mag = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
    assert bool(((y - want).abs() <= (k + 16) * R.U32 * mag + 2.0 ** -149 * k).all())
    for rows, cols in ((slice(300, 310), slice(6, n)), (slice(0, 300), slice(5, 6)), (slice(0, 300), slice(6, n))):
        a, b = y[rows, cols], want[rows, cols]
        a, b = a / b.abs().max(), b / b.abs().max()
        assert float((a - b).square().mean().sqrt() / b.square().mean().sqrt()) <= R.U32 * k ** 0.5, (rows, cols)
    assert float(y[700:800].abs().max()) == 0


def tails(dt, act, slope=0.0):
    """act and act' where they are small next to 1, one value a row: -> ((y, its value, the sum of its terms' magnitudes), the same of act')."""
    s = torch.linspace(-12.5, 12.5, 6001).to(dt)[:, None]
    one = torch.ones(1, 1, dtype=dt)
    y = ops.linear(s.to(dev()), one.to(dev()), None, act, slope).cpu().double()
    got, _ = gradients(s, one, None, act, torch.ones_like(s), slope)
    S = s.double()
    sig, sig_ = torch.special.expit(S), torch.special.expit(-S)
    if act == "gelu":
        cdf, pdf = torch.special.erfc(-S / 2 ** 0.5) / 2, torch.exp(-S * S / 2) / (2 * torch.pi) ** 0.5
        v, d, mag = S * cdf, cdf + S * pdf, cdf + S.abs() * pdf
    elif act == "sigmoid":
        v, d, mag = sig, sig * sig_, sig * sig_
    elif act == "silu":
        v, d, mag = S * sig, sig * (1 + S * sig_), sig * (1 + S.abs() * sig_)
    else:
        d = 4 * torch.exp(-2 * S.abs()) / (1 + torch.exp(-2 * S.abs())) ** 2
        v, mag = torch.tanh(S), d
    return S, (y, v, v.abs()), (got["dx"].cpu().double(), d, mag)


def check_tails(dt, act, rel):
    """rel(s): the relative error that the evaluation may have; the result's own rounding comes on top."""
    S, *both = tails(dt, act)
    for name, (got, want, mag) in zip(("y", "slope"), both):
        bound = R.u(dt) * want.abs() + rel(S) * mag + R.tiny(dt) + 2.0 ** -126
        err = (got - want).abs()
        assert bool((err <= bound).all()), (name, float((err / bound).max()), float(S[(err / bound).argmax()]))


# exp's argument is rounded, which moves the result by |argument| half steps for each of its roundings; 16 half steps for the rest
@pytest.mark.parametrize("dt", R.DTYPES)
def test_gelu_keeps_its_digits_in_the_tail(dt):
    """exp(-s^2 / 2) and erfc(-s / sqrt 2), whose argument is rounded twice and counts twice: 3 s^2 half steps.  (16-bit results: a polynomial
    with a relative error of 2^-22 more.)"""
    check_tails(dt, "gelu", lambda s: (16 + 3 * s * s) * R.U32 + (2.0 ** -22 if dt != F32 else 0.0))


@pytest.mark.parametrize("act", ["sigmoid", "xtanh", "silu"])
@pytest.mark.parametrize("dt", R.DTYPES)
def test_slopes_keep_their_digits_in_the_tails(dt, act):
    """exp(-s) and exp(-2 |s|): 2 |s| half steps, twice (argument and constant)."""
    check_tails(dt, act, lambda s: (16 + 4 * s.abs()) * R.U32 + (2.0 ** -18 if act == "xtanh" and dt != F32 else 0.0))


@pytest.mark.parametrize("off", [0, 1, 5])
@pytest.mark.parametrize("dt", R.DTYPES)
def test_residual_rows_at_any_offset_of_a_large_product(dt, off):
    """The residual's rows start anywhere, the first and the last of them at the ends of the allocation."""
    g = torch.Generator().manual_seed(10)
    m, k, n = 4100, 520, 2003
    x, w, r = (torch.randint(-3, 4, s, generator=g).to(dt).to(dev()) for s in ((m, k), (n, k), (m, n)))
    if dt != F32:       # a large product whose sums are not split needs no workspace here; it is these that bring the residual into the cache
        assert ops._linear_plan(m, k, n, ops.DTYPE_IDS[dt], 0, R.SLOPE, k, n, 0, 0)[1] == 0
    for ld in (n, n + 6, n + 7):
        flat = torch.full((off + (m - 1) * ld + n,), float("nan"), dtype=dt, device=dev())
        view = flat[off:].as_strided((m, n), (ld, 1))
        view.copy_(r)
        assert torch.equal(ops.linear(x, w, residual=view), (x.double() @ w.double().t() + r.double()).to(dt))
