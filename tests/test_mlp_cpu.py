"""MLP's operator path without a GPU."""
import io

import torch

from ivae_amd import MLP


def test_mlp_pickled_before_the_options_still_runs():
    """An MLP object stored whole by a version without layer_norm, residual and dropout lacks their attributes."""
    torch.manual_seed(0)
    m = MLP(3, 2, 8, 3, activation="lrelu")
    x = torch.randn(4, 3)
    want = m(x)
    for name in ("residual", "dropout", "operators"):
        m.__dict__.pop(name, None)
    m.__dict__.pop("norm", None), m._modules.pop("norm", None)
    f = io.BytesIO()
    torch.save(m, f)
    f.seek(0)
    old = torch.load(f, weights_only=False)         # (this test's own file)
    assert torch.equal(old(x), want) and torch.equal(old.eval()(x), want)
