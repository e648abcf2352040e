"""What the tensor operators refuse, without a GPU: the C entries' codes, the Python checks, and the oracle itself."""
import ctypes as C
import os
import shutil
import subprocess

import pytest
import torch

from ivae_amd import MLP, _lib, ops
from tests import operator_ref as R


def test_philox_known_answers():
    """The three vectors published with Philox4x32-10 (Random123's kat_vectors), through the mask's threshold: the oracle's words
    are compared one by one with the published ones."""
    import numpy as np

    def words(ctr, key):
        # counter word 0/1 = element / 4, 2/3 = offset; read the words by bisecting nothing: rebuild them from keep() at 32 thresholds
        q = ctr[0] | ctr[1] << 32
        seed, offset = key[0] | key[1] << 32, ctr[2] | ctr[3] << 32
        assert q == 0
        out = [0, 0, 0, 0]
        for bit in range(31, -1, -1):
            for j in range(4):
                trial = out[j] | 1 << bit
                if bool(R.keep(4, trial / 2 ** 32, seed, offset)[j]):
                    out[j] = trial
        return out
    assert words((0, 0, 0, 0), (0, 0)) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    assert np.array_equal(R.keep(8, 0.5, 0, 0)[:4].numpy(), np.array([0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]) >= 2 ** 31)


@pytest.mark.parametrize("act", R.ACTS)
def test_formulas_against_differences(act):
    """The oracle's gradients against central differences of its values, in 64 bits: the truncation is h^2 |third derivative| / 6
    (under 1e-9 at h = 1e-5 for these sizes), the cancellation 1e-16 / h."""
    g = torch.Generator().manual_seed(1)
    x, w, b, dy = (torch.randn(*s, generator=g, dtype=torch.float64).float() for s in ((5, 7), (6, 7), (6,), (5, 6)))
    o = R.linear64(x, w, b, act, None, dy)
    f = lambda X, W, B: float((R.act64(X @ W.t() + B, act)[0] * dy.double()).sum())  # noqa: E731
    h = 1e-5
    for name, t, i in (("dx", x, 0), ("dw", w, 1), ("db", b, 2)):
        d = torch.randn(t.shape, generator=g, dtype=torch.float64)
        args = [x.double(), w.double(), b.double()]
        up, dn = list(args), list(args)
        up[i], dn[i] = args[i] + h * d, args[i] - h * d
        assert abs((f(*up) - f(*dn)) / (2 * h) - float((o[name][0] * d).sum())) < 1e-6


def test_norm_formula_against_differences():
    g = torch.Generator().manual_seed(2)
    x, w, b, dy = (torch.randn(*s, generator=g) for s in ((4, 9), (9,), (9,), (4, 9)))
    o = R.norm64(x, w, b, 1e-5, dy)
    f = lambda X, W, B: float((torch.nn.functional.layer_norm(X, (9,), W, B, 1e-5) * dy.double()).sum())  # noqa: E731
    for name, i in (("dx", 0), ("dw", 1), ("db", 2)):
        args = [x.double(), w.double(), b.double()]
        d = torch.randn(args[i].shape, generator=g, dtype=torch.float64)
        up, dn = list(args), list(args)
        up[i], dn[i] = args[i] + 1e-5 * d, args[i] - 1e-5 * d
        assert abs((f(*up) - f(*dn)) / 2e-5 - float((o[name][0] * d).sum())) < 1e-6


# ---- C entries: every refusal comes back as a code before anything is launched ----------------------------------------

P = C.c_void_p(64)      # never dereferenced: each of these calls is refused before a launch


def _lin(rows=4, k=8, n=8, dtype=0, act=0, ldx=8, ldr=8, lddy=8):
    return _lib.IvaeLinear(rows, k, n, dtype, act, .1, ldx, ldr, lddy)


@pytest.mark.parametrize("kw,code", [(dict(rows=-1), -1), (dict(k=0), -1), (dict(n=0), -1), (dict(ldx=-1), -1), (dict(ldr=-8), -1), (dict(lddy=-1), -1),
                                     (dict(dtype=3), -7), (dict(dtype=-1), -7), (dict(act=6), -2), (dict(act=-1), -2),
                                     (dict(k=(1 << 24) + 1), -4), (dict(n=(1 << 24) + 1), -4), (dict(rows=(1 << 40) + 1), -4)])
def test_linear_refuses(kw, code):
    L = _lib.lib()
    nb = C.c_size_t()
    lin = _lin(**kw)
    assert L.ivae_linear_workspace_bytes(lin, 0, C.byref(nb)) == code
    assert L.ivae_linear(lin, P, P, P, P, P, P, P, 1 << 40, None) == code
    assert L.ivae_linear_backward(lin, P, P, P, P, P, P, P, P, 1 << 40, None) == code


def test_linear_refuses_missing_pointers_and_small_workspaces():
    L = _lib.lib()
    nb = C.c_size_t()
    assert L.ivae_linear_workspace_bytes(None, 0, C.byref(nb)) == -3 and L.ivae_linear_workspace_bytes(_lin(), 0, None) == -3
    for hole in range(3):
        args = [P, P, P]                                  # x, w, y
        args[hole] = None
        assert L.ivae_linear(_lin(), args[0], args[1], None, None, args[2], None, None, 0, None) == -3
    assert L.ivae_linear(None, P, P, None, None, P, None, None, 0, None) == -3
    assert L.ivae_linear_backward(_lin(), None, P, P, None, P, P, P, None, 0, None) == -3
    assert L.ivae_linear_backward(_lin(), P, None, P, None, P, P, P, None, 0, None) == -3
    assert L.ivae_linear_backward(_lin(), P, P, None, None, P, P, P, None, 0, None) == -3
    assert L.ivae_linear_backward(_lin(act=1), P, P, P, None, P, P, P, None, 0, None) == -3       # an activation without `saved`
    lin = _lin(rows=4, k=4096, n=64, ldx=4096)
    assert L.ivae_linear_workspace_bytes(lin, 0, C.byref(nb)) == 0 and nb.value > 0
    assert L.ivae_linear(lin, P, P, None, None, P, None, None, nb.value, None) == -3
    assert L.ivae_linear(lin, P, P, None, None, P, None, P, nb.value - 1, None) == -6
    assert L.ivae_linear(_lin(rows=0), P, P, None, None, P, None, None, 0, None) == 0             # nothing to do


@pytest.mark.parametrize("kw,code", [(dict(rows=-1), -1), (dict(width=0), -1), (dict(ldx=-1), -1), (dict(lddy=-1), -1), (dict(ldr=-1), -1),
                                     (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1), (dict(dtype=7), -7), (dict(width=(1 << 24) + 1), -4),
                                     (dict(rows=(1 << 40) + 1), -4)])
def test_layer_norm_refuses(kw, code):
    L = _lib.lib()
    a = dict(dict(rows=4, width=8, dtype=0, w32=1, eps=1e-5, ldx=8, lddy=8, ldr=8), **kw)
    norm = _lib.IvaeNorm(a["rows"], a["width"], a["dtype"], a["w32"], a["eps"], a["ldx"], a["lddy"], a["ldr"])
    nb = C.c_size_t()
    assert L.ivae_layer_norm_workspace_bytes(norm, C.byref(nb)) == code
    assert L.ivae_layer_norm(norm, P, P, P, P, P, None) == code
    assert L.ivae_layer_norm_backward(norm, P, P, P, P, P, P, P, P, P, 1 << 40, None) == code


def test_layer_norm_refuses_missing_pointers_and_small_workspaces():
    L = _lib.lib()
    nb = C.c_size_t()
    # the gradients of few rows need no workspace
    few = _lib.IvaeNorm(4, 8, 0, 1, 1e-5, 8, 8, 8)
    assert L.ivae_layer_norm_workspace_bytes(few, C.byref(nb)) == 0 and nb.value == 0
    norm = _lib.IvaeNorm(400, 8, 0, 1, 1e-5, 8, 8, 8)
    assert L.ivae_layer_norm_workspace_bytes(norm, C.byref(nb)) == 0 and nb.value > 0
    assert L.ivae_layer_norm(norm, None, P, P, P, P, None) == -3 and L.ivae_layer_norm(norm, P, P, P, None, P, None) == -3
    for hole in range(3):
        args = [P, P, P]
        args[hole] = None
        assert L.ivae_layer_norm_backward(norm, *args, P, None, P, P, P, P, nb.value, None) == -3
    assert L.ivae_layer_norm_backward(norm, P, P, P, P, None, P, P, P, None, nb.value, None) == -3
    assert L.ivae_layer_norm_backward(norm, P, P, P, P, None, P, P, P, P, nb.value - 1, None) == -6
    assert L.ivae_layer_norm_backward(None, P, P, P, P, None, P, P, P, P, 0, None) == -3


def test_dropout_refuses():
    L = _lib.lib()
    assert L.ivae_dropout(5, 8, P, None, P, .1, 0, 0, None, None) == -7
    assert L.ivae_dropout(0, -1, P, None, P, .1, 0, 0, None, None) == -1
    for p in (-0.1, 1.5, float("nan")):
        assert L.ivae_dropout(0, 8, P, None, P, p, 0, 0, None, None) == -1
    assert L.ivae_dropout(0, 8, None, None, P, .1, 0, 0, None, None) == -3 and L.ivae_dropout(0, 8, P, None, None, .1, 0, 0, None, None) == -3
    assert L.ivae_dropout(0, 0, None, None, None, .1, 0, 0, None, None) == 0


# ---- Python checks ----------------------------------------------------------------------------------------------------


def test_operators_need_a_device():
    x, w = torch.zeros(2, 3), torch.zeros(4, 3)
    for call in (lambda: ops.linear(x, w), lambda: ops.linear_backward(torch.zeros(2, 4), x, w), lambda: ops.layer_norm(x),
                 lambda: ops.layer_norm_backward(x, x, torch.zeros(2, 2)), lambda: ops.dropout(x, .1, 0)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    for call in (lambda: ops.linear(x.double(), w), lambda: ops.layer_norm(x.double()), lambda: ops.dropout(x.long(), .1, 0)):
        with pytest.raises(TypeError):
            call()


def test_mlp_options():
    plain = MLP(3, 2, 8, 3, activation="lrelu")
    assert not plain.operators and list(plain.state_dict()) == [f"fc.{i}.{n}" for i in range(3) for n in ("weight", "bias")]
    m = MLP(3, 2, 8, 3, activation="gelu", layer_norm=True, residual=True, dropout=.1)
    assert [k for k in m.state_dict() if k.startswith("norm")] == ["norm.0.weight", "norm.0.bias", "norm.1.weight", "norm.1.bias"]
    with pytest.raises(RuntimeError, match="no CPU path"):
        m(torch.zeros(4, 3))
    with pytest.raises(ValueError):
        MLP(3, 2, 8, 3, activation="gelu")               # the torch path keeps the reference's activations
    with pytest.raises(ValueError):
        MLP(3, 2, 8, 3, dropout=1.5)


ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(not (shutil.which("hipcc") or os.path.exists("/opt/rocm/bin/hipcc")), reason="needs hipcc to build")
def test_host_paths_are_clean_under_asan_and_ubsan():
    """Every choice that the host makes for a call (kernel, tiles, splits, pieces of the workspace), over random shapes, instrumented."""
    b = subprocess.run(["make", "-j8", "build/abi_asan_ops"], cwd=ROOT, capture_output=True, text=True, timeout=900)
    assert b.returncode == 0, b.stdout[-2000:] + b.stderr[-2000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:abort_on_error=0", UBSAN_OPTIONS="print_stacktrace=1")
    r = subprocess.run([os.path.join(ROOT, "build", "abi_asan_ops")], cwd=ROOT, capture_output=True, text=True, timeout=600, env=env)
    assert r.returncode == 0 and "abi_asan_ops: OK" in r.stdout, r.stdout[-2000:] + r.stderr[-4000:]
