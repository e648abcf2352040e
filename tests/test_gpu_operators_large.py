"""The large kernels of linear, at sizes that tests/test_operator_shapes_cpu.py holds to reach them: every instance on whole numbers, every
activation and layout against the formulas in 64 bits, and that nothing beyond the results is written."""
import pytest
import torch

from ivae_amd import _lib, ops
from tests import operator_ref as R
from tests import operator_shapes as S
from tests.test_gpu_operators import dev, normal, run_linear

pytestmark = pytest.mark.gpu


def whole(g, *shape, dtype, top=3):
    return torch.randint(-top, top + 1, shape, generator=g).to(dtype).to(dev())


@pytest.mark.parametrize("m,k,n", S.BOTH)
@pytest.mark.parametrize("dt", R.DTYPES)
def test_whole_numbers_are_exact_and_nothing_beyond_is_written(dt, m, k, n):
    """Sums of whole numbers below 2^24, each rounded once to its type.  Every buffer ends in values that have to stay, the workspace too."""
    g = torch.Generator().manual_seed(m + k + n)
    x, w, dy, r = (whole(g, *s, dtype=dt) for s in ((m, k), (n, k), (m, n), (m, n)))
    b = whole(g, n, dtype=dt, top=9)
    X, W, D = x.double(), w.double(), dy.double()
    s = X @ W.t() + b.double()
    stream, L, code = torch.cuda.current_stream().cuda_stream, _lib.lib(), ops.DTYPE_IDS[dt]

    def guarded(count, dtype):
        t = torch.full((count + 4096,), 7.0, dtype=dtype, device=dev())
        return t, t.data_ptr()
    for act, slope in (("none", .1), ("lrelu", 2.0)):
        k2 = torch.where(s > 0, 1.0, 2.0) if act == "lrelu" else torch.ones_like(s)
        ds = D * k2
        want = {"y": s * k2 + r.double(), "dx": ds @ W, "dw": ds.t() @ X, "db": ds.sum(0)}
        bufs = {"y": guarded(m * n, dt), "saved": guarded(m * n, torch.float32), "dx": guarded(m * k, dt), "dw": guarded(n * k, dt), "db": guarded(n, dt)}
        for backward in (0, 1):
            lin, nb = ops._linear_plan(m, k, n, code, _lib.LINEAR_ACT_IDS[act], slope, k, n, n, backward)
            ws = torch.full((nb + 4096,), 7, dtype=torch.uint8, device=dev())
            if backward:
                rc = L.ivae_linear_backward(lin, dy.data_ptr(), x.data_ptr(), w.data_ptr(), bufs["saved"][1], bufs["dx"][1], bufs["dw"][1], bufs["db"][1],
                                            ws.data_ptr(), nb, stream)
            else:
                rc = L.ivae_linear(lin, x.data_ptr(), w.data_ptr(), b.data_ptr(), r.data_ptr(), bufs["y"][1], bufs["saved"][1] if act != "none" else None,
                                   ws.data_ptr(), nb, stream)
            assert rc == 0 and bool((ws[nb:] == 7).all()), (act, backward)
        for name, v in want.items():
            t = bufs[name][0]
            assert torch.equal(t[:v.numel()].view(v.shape), v.to(dt)), (act, name)
        if act != "none":
            assert torch.equal(bufs["saved"][0][:m * n].view(m, n), s.float())
        assert all(bool((t[-4096:] == 7).all()) for t, _ in bufs.values())


@pytest.mark.parametrize("act", R.ACTS)
@pytest.mark.parametrize("dt", R.DTYPES)
def test_activations(dt, act):
    run_linear(dt, 2050, 1100, 1201, act, seed=3)


@pytest.mark.parametrize("layout", ["strided", "transposed"])
@pytest.mark.parametrize("act", ["none", "xtanh", "sigmoid"])
@pytest.mark.parametrize("dt", R.DTYPES)
def test_layouts(dt, act, layout):
    """x, the residual and dy with rows at an odd offset of wider ones, amid NaN; x, w and dy transposed."""
    run_linear(dt, 1100, 1501, 1003, act, layout=layout, seed=4)
    run_linear(dt, 4100, 520, 2003, act, layout=layout, bias=False, res=layout == "strided", seed=5)


@pytest.mark.parametrize("dt", R.DTYPES)
@pytest.mark.parametrize("need", [(True, False, False), (False, True, False), (False, False, True), (False, True, True), (True, False, True)])
def test_parts_of_the_gradients(dt, need):
    for act in ("none", "gelu"):
        full = run_linear(dt, 1100, 1501, 1003, act, seed=6)
        part = run_linear(dt, 1100, 1501, 1003, act, seed=6, need=need)
        assert all(b is None or torch.equal(a, b) for a, b in zip(full[-1], part[-1]))


@pytest.mark.parametrize("dt", R.DTYPES)
@pytest.mark.parametrize("m,k,n", [(2050, 1100, 1201), (300, 1100, 9000)])
def test_misaligned(dt, m, k, n):
    """Dense matrices that start one element off a 16-byte boundary."""
    g = torch.Generator().manual_seed(7)
    mats = []
    for shape in ((m, k), (n, k), (m, n), (m, n)):
        flat = torch.empty(shape[0] * shape[1] + 1, dtype=dt, device=dev())
        flat[1:].view(shape).copy_(whole(g, *shape, dtype=dt))
        mats.append(flat[1:].view(shape))
    x, w, dy, r = mats
    X, W, D = x.double(), w.double(), dy.double()
    assert torch.equal(ops.linear(x, w, residual=r), (X @ W.t() + r.double()).to(dt))
    for got, want in zip(ops.linear_backward(dy, x, w), (D @ W, D.t() @ X, D.sum(0))):
        assert torch.equal(got, want.to(dt))


@pytest.mark.parametrize("dt", R.DTYPES)
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_replays_and_streams(dt, act):
    """A step captured into a graph and replayed, eager work between, and the same step on another stream: the eager call's bits."""
    g = torch.Generator().manual_seed(8)
    m, k, n = 1100, 1501, 1003
    x, w, dy = (normal(g, *s, scale=.2, dtype=dt).to(dev()) for s in ((m, k), (n, k), (m, n)))

    def step():
        y, saved = ops.linear(x, w, None, act, residual=dy, save=True)
        return y, *ops.linear_backward(dy, x, w, saved, act)
    want = [t.clone() for t in step()]
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        out = step()
    for _ in range(3):
        for t in out:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        other = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, out, other))


@pytest.mark.parametrize("dt", R.DTYPES)
def test_repeated_and_overlapping_rows(dt):
    """x one row repeated (stride 0), rows that overlap by all but one element (stride 1), x as the residual, and dy as x."""
    g = torch.Generator().manual_seed(9)
    m, k = 2200, 1104
    w = whole(g, k, k, dtype=dt)
    flat = whole(g, m + k, dtype=dt)
    for x in (flat[:k].expand(m, k), flat.as_strided((m, k), (1, 1)), flat.as_strided((m, k), (0, 1))):
        X, W = x.double(), w.double()
        assert S.plan(m, k, k, ops.DTYPE_IDS[dt])[0] == S.LARGE
        assert torch.equal(ops.linear(x, w, residual=x), (X @ W.t() + X).to(dt))
        for got, want in zip(ops.linear_backward(x, x, w), (X @ W, X.t() @ X, X.sum(0))):
            assert torch.equal(got, want.to(dt))
