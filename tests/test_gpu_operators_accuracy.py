"""How exact the tensor operators are where worst-case bounds of long sums see nothing: root mean squares of errors against the rounding
of the results alone, values at the ends of a type's range, infinities that meet a zero of a split value."""
import pytest
import torch

from ivae_amd import ops
from tests import operator_ref as R

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
# one product that the 64 x 64 kernel takes, one that the large kernels take, and one of odd sizes
SIZES = [(96, 120, 104), (1024, 768, 520), (1003, 777, 531)]
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
