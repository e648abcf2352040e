"""Drop-in model classes for the reference's ``models/nets.py`` hot path.

Same constructors, ``forward`` / ``elbo`` / ``anneal`` signatures and ``state_dict`` keys as
``MLP`` (nets.py:65-121), ``cleanIVAE`` (124-185), ``cleanVAE`` (188-243), ``Normal``
(293-314), ``iVAE`` (391-486) and ``VAE`` (548-599), so ``runners/ivae.py`` and
``models/wrappers.py`` can import them unchanged.  The arithmetic of ``forward`` and ``elbo``
(+ its backward) runs in libivae_amd.so's HIP kernels through ``ivae_amd.ops``; the modules
only own parameters (ordinary ``nn.Parameter`` views into one flat fp32 arena) and scalars.
There is no CPU path: calling ``forward``/``elbo`` off a ROCm device raises.
"""
from numbers import Number

import numpy as np
import torch
from torch import nn
from torch.autograd.function import once_differentiable
from torch.nn import functional as F

from . import ops
from .ops import ModelShape


def weights_init(m):
    """nets.py:10-12."""
    if isinstance(m, nn.Linear):
        nn.init.xavier_uniform_(m.weight.data)


class Normal:
    """Marker for the only distribution the fused path implements (nets.py:293-314).
    ``sample``/``log_pdf`` are kept for callers that use them directly (plain torch ops)."""
    name = 'gauss'

    def __init__(self, device='cpu'):
        self.device = device
        self.c = 2 * np.pi * torch.ones(1).to(self.device)

    def sample(self, mu, v):
        eps = torch.randn_like(mu)
        return eps.mul(v.sqrt()).add(mu)

    def log_pdf(self, x, mu, v, reduce=True, param_shape=None):
        if param_shape is not None:
            mu, v = mu.view(param_shape), v.view(param_shape)
        lpdf = -0.5 * (torch.log(self.c) + v.log() + (x - mu).pow(2).div(v))
        return lpdf.sum(dim=-1) if reduce else lpdf


def _no_capture(*tensors):
    """The autograd engine synchronises the streams of a graph's leaves by itself, which a capture on another stream does not
    survive: gradients under capture are the business of ``ops`` (``linear_backward`` and its siblings capture like any launch)."""
    if any(t is not None and t.is_cuda for t in tensors) and torch.cuda.is_current_stream_capturing():
        raise RuntimeError('autograd through MLP operators cannot be captured into a graph: capture ivae_amd.ops calls instead')


# The operators go through these Functions without gradients as well: forward mode and tracing know nothing of what runs outside of one,
# and would drop it in silence.  Inside a Function its caller's grad mode is not to be seen, so `grad` says whether to keep anything.
class _LinearFn(torch.autograd.Function):
    """ops.linear with its gradients."""

    @staticmethod
    def forward(ctx, x, weight, bias, activation, slope, residual, grad):
        if not (grad and any(ctx.needs_input_grad[:3])):
            return ops.linear(x, weight, bias, activation, slope, residual)
        _no_capture(x)
        y, pre = ops.linear(x, weight, bias, activation, slope, residual, save=True)
        ctx.save_for_backward(x, weight, pre)
        ctx.act = activation, slope
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _no_capture(dy)
        need = ctx.needs_input_grad
        dx = dw = db = None
        if any(need[:3]):
            x, weight, pre = ctx.saved_tensors
            dx, dw, db = ops.linear_backward(dy, x, weight, pre, *ctx.act, need=need[:3])
        return dx, dw, db, None, None, dy if need[5] else None, None


class _LayerNormFn(torch.autograd.Function):
    """ops.layer_norm with its gradients."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps, grad):
        if not (grad and any(ctx.needs_input_grad[:3])):
            return ops.layer_norm(x, weight, bias, eps)
        _no_capture(x)
        y, stats = ops.layer_norm(x, weight, bias, eps, save=True)
        ctx.save_for_backward(x, weight, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _no_capture(dy)
        x, weight, stats = ctx.saved_tensors
        return (*ops.layer_norm_backward(dy, x, stats, weight, need=ctx.needs_input_grad[:3]), None, None)


class _DropoutFn(torch.autograd.Function):
    """ops.dropout with its gradients; the mask is drawn again in the backward pass."""

    @staticmethod
    def forward(ctx, x, p, seed, offset, residual, grad):
        if grad and any(ctx.needs_input_grad):
            _no_capture(x)
        ctx.draw = p, seed, offset
        return ops.dropout(x, p, seed, offset, residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _no_capture(dy)
        need = ctx.needs_input_grad
        return ops.dropout_backward(dy, *ctx.draw) if need[0] else None, None, None, None, dy if need[4] else None, None


class _OperatorLinear(nn.Linear):
    """nn.Linear on ops.linear, with the activation and the residual that its caller passes fused into it."""

    def forward(self, x, activation='none', slope=.1, residual=None):
        return _LinearFn.apply(x, self.weight, self.bias, activation, slope, residual, torch.is_grad_enabled())


class _OperatorNorm(nn.LayerNorm):
    """nn.LayerNorm over the last dimension on ops.layer_norm."""

    def forward(self, x):
        return _LayerNormFn.apply(x, self.weight, self.bias, self.eps, torch.is_grad_enabled())


def _fuses(fc):
    """Whether what follows fc may run inside it: it is this module's own, and nobody asked for its output or its gradients."""
    return isinstance(fc, _OperatorLinear) and not (fc._forward_hooks or fc._backward_hooks or fc._backward_pre_hooks)


class MLP(nn.Module):
    """Container with the reference's constructor and ``fc`` ModuleList (nets.py:66-107).
    Inside the fused models only its parameters are used; its own ``forward`` (plain torch
    ops) exists for callers that evaluate a sub-network by itself.

    ``layer_norm``, ``residual`` and ``dropout`` (no counterpart in the reference) turn the hidden layers into residual blocks,
    ``h + dropout(act(fc(norm(h))))``: every layer but the first normalises its input (``norm.<layer - 1>``), the sum is taken where a
    hidden layer's two widths agree, and dropout acts in training mode, its seed drawn from torch's CPU generator.  With any of
    them the forward and backward passes run in the library's kernels (``ops.linear``, ``ops.layer_norm``, ``ops.dropout``) and need
    a ROCm device; fp32, bf16 and fp16 parameters, and the activations 'gelu' and 'silu' besides the others.  ``fc`` and ``norm`` hold
    modules that are called, so hooks run, and what rebuilds a weight before a call (weight norm, spectral norm, pruning) acts; where an
    ``fc`` has forward or backward hooks or was replaced, its activation and the sum run in torch, outside of it."""

    operators = False           # of an MLP that was pickled before there were these options

    def __init__(self, input_dim, output_dim, hidden_dim, n_layers, activation='none', slope=.1, device='cpu', layer_norm=False,
                 residual=False, dropout=0.):
        super().__init__()
        if not 0. <= dropout <= 1.:
            raise ValueError('dropout must be between 0 and 1: {}'.format(dropout))
        self.residual = bool(residual)
        self.dropout = float(dropout)
        self.operators = bool(layer_norm or residual or dropout)
        self.input_dim = input_dim
        self.output_dim = output_dim
        self.n_layers = n_layers
        self.device = device
        self.slope = slope
        if isinstance(hidden_dim, Number):
            self.hidden_dim = [hidden_dim] * (self.n_layers - 1)
        elif isinstance(hidden_dim, list):
            self.hidden_dim = hidden_dim
        else:
            raise ValueError('Wrong argument type for hidden_dim: {}'.format(hidden_dim))
        if isinstance(activation, str):
            self.activation = [activation] * (self.n_layers - 1)
        elif isinstance(activation, list):
            self.activation = activation
        else:
            raise ValueError('Wrong argument type for activation: {}'.format(activation))
        for act in self.activation:
            if act not in (ops.LINEAR_ACT_IDS if self.operators else ops.ACT_IDS):
                raise ValueError('Incorrect activation: {}'.format(act))
        dims = [self.input_dim] + list(self.hidden_dim[:self.n_layers - 1]) + [self.output_dim]
        linear = _OperatorLinear if self.operators else nn.Linear
        self.fc = nn.ModuleList([linear(dims[i], dims[i + 1]) for i in range(self.n_layers)])
        self.norm = nn.ModuleList([_OperatorNorm(d) for d in dims[1:-1]]) if layer_norm else None
        self.to(self.device)

    @staticmethod
    def xtanh(x, alpha=.1):
        return x.tanh() + alpha * x

    def _act(self, kind, h):
        if kind == 'lrelu':
            return F.leaky_relu(h, negative_slope=self.slope)
        if kind == 'xtanh':
            return self.xtanh(h, alpha=self.slope)
        if kind == 'sigmoid':
            return torch.sigmoid(h)
        if kind == 'gelu':
            return F.gelu(h)
        if kind == 'silu':
            return F.silu(h)
        return h

    def _forward_operators(self, x):
        if not x.is_cuda:
            raise RuntimeError('x must live on a ROCm device: ivae_amd has no CPU path')
        drop = self.dropout if self.training else 0.
        seed = 0
        if drop:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError('a captured MLP would draw the same dropout mask at every replay: call eval() first')
            if torch.jit.is_tracing():
                raise RuntimeError('a traced MLP would draw the same dropout mask at every call: call eval() first')
            seed = int(torch.randint(2 ** 63 - 1, ()))
        h = x
        for c, fc in enumerate(self.fc):
            t = self.norm[c - 1](h) if self.norm is not None and c else h
            if c == self.n_layers - 1:
                return fc(t)
            # (the sum joins a layer whose result has its input's width)
            fused = _fuses(fc)
            if fused:
                add = h if self.residual and fc.in_features == fc.out_features else None
                t = fc(t, self.activation[c], self.slope, None if drop else add)
            else:
                t = self._act(self.activation[c], fc(t))
                add = h if self.residual and t.shape[-1] == h.shape[-1] else None
            if drop:
                t = _DropoutFn.apply(t, drop, seed, c, add, torch.is_grad_enabled())
            elif add is not None and not fused:
                t = t + add
            h = t
        return h

    def forward(self, x):
        if self.operators:
            return self._forward_operators(x)
        h = x
        for c in range(self.n_layers):
            h = self.fc[c](h)
            if c != self.n_layers - 1:
                h = self._act(self.activation[c], h)
        return h


class _ElboFn(torch.autograd.Function):
    """One fused launch sequence computes loss, z and every parameter gradient; backward only
    scales the stashed flat gradient by the incoming scalar (runners/ivae.py:82 passes 1,
    wrappers.py:69 passes -1 through ``elbo.mul(-1)``)."""

    @staticmethod
    def forward(ctx, model, coef, x, u, eps, *params):
        loss, z, grads = ops.elbo_fwd_bwd(model._shape, coef, model._flat_params(), x, u, eps, model._ws)
        ctx.flat_grads = grads
        ctx.sizes = [p.numel() for p in params]
        ctx.shapes = [p.shape for p in params]
        ctx.mark_non_differentiable(z)
        return loss[0], z

    @staticmethod
    def backward(ctx, gl, gz):
        flat = ctx.flat_grads * gl
        outs, off = [], 0
        for n, s in zip(ctx.sizes, ctx.shapes):
            outs.append(flat[off:off + n].view(s))
            off += n
        return (None, None, None, None, None) + tuple(outs)


class _FusedModel(nn.Module):
    """Shared machinery: flat parameter arena, workspace, kernel dispatch."""

    def _finish_init(self, data_dim, latent_dim, aux_dim, hidden_dim, n_layers, activation, slope):
        if not isinstance(hidden_dim, Number) or not isinstance(activation, str):
            raise NotImplementedError('the fused path supports one hidden width and one activation for all layers')
        self._shape = ModelShape(int(data_dim), int(latent_dim), int(aux_dim), int(hidden_dim), int(n_layers),
                                 activation, float(slope))
        self._ws = ops.Workspace()
        self._arena = None
        self._pack()

    # -- parameter arena -------------------------------------------------------------
    def _pack(self):
        ps = list(self.parameters())
        total = sum(p.numel() for p in ps)
        arena = torch.empty(total, dtype=ps[0].dtype, device=ps[0].device)
        off = 0
        with torch.no_grad():
            for p in ps:
                n = p.numel()
                arena[off:off + n].copy_(p.data.reshape(-1))
                p.data = arena[off:off + n].view(p.shape)
                off += n
        self._arena = arena

    def _apply(self, fn, *args, **kwargs):
        out = super()._apply(fn, *args, **kwargs)
        if getattr(self, '_shape', None) is not None:
            self._pack()
        return out

    def _flat_params(self):
        """The arena, re-packed first if some parameter no longer aliases it."""
        off = 0
        base = self._arena.data_ptr()
        for p in self.parameters():
            if p.data_ptr() != base + 4 * off or p.device != self._arena.device:
                self._pack()
                break
            off += p.numel()
        if self._arena.dtype != torch.float32:
            raise TypeError('ivae_amd kernels are fp32 only')
        return self._arena

    # -- kernels ---------------------------------------------------------------------
    def _eps(self, x, eps):
        """The draw of nets.py:147 / nets.py:302 (torch.randn), on the inputs' device."""
        if eps is None:
            eps = torch.randn(x.shape[0], self._shape.latent_dim, dtype=torch.float32, device=x.device)
        return eps

    FORWARD_ROWS = 65536     # rows per ivae_forward call: a full-dataset forward (runners/ivae.py:118-122) runs in blocks

    def _forward_tensors(self, x, u, eps=None):
        sh = self._shape
        eps = self._eps(x, eps)
        B = x.shape[0]
        params = self._flat_params()
        mk = lambda w: torch.empty(B, w, dtype=torch.float32, device=x.device)
        f, g, v, l, z = mk(sh.data_dim), mk(sh.latent_dim), mk(sh.latent_dim), mk(sh.latent_dim), mk(sh.latent_dim)
        # every row's forward is independent of the others, so blocks give the same values as one call; the workspace
        # (hidden activations of every layer) stays bounded for N = 1e6-row datasets
        for lo in range(0, B, self.FORWARD_ROWS):
            hi = min(B, lo + self.FORWARD_ROWS)
            n = hi - lo
            coef = ops.make_coef(decoder_var=self._decoder_var_f, global_batch=n)
            z[lo:hi] = ops.forward(sh, coef, params, x[lo:hi], None if u is None else u[lo:hi], eps[lo:hi], self._ws)
            g[lo:hi] = self._ws.view('g', n, sh.latent_dim)
            v[lo:hi] = self._ws.view('v', n, sh.latent_dim)
            l[lo:hi] = self._ws.view('l', n, sh.latent_dim)
            f[lo:hi] = self._ws.view('f', n, sh.data_dim)
        return f, g, v, z, l

    def direct_step(self, optimizer, x, u, a, b, c, d, N, pairwise, eps=None, z_out=None):
        """zero_grad -> elbo -> backward -> optimizer.step() (runners/ivae.py:75-91) without the autograd and
        per-parameter optimizer machinery: ivae_elbo_fwd_bwd writes the flat gradient, `optimizer.step_flat`
        (ivae_amd.FusedAdam) consumes it.  Same kernels, same noise draw, same update as the drop-in sequence.
        Returns (loss, z) like `elbo` (loss detached)."""
        eps = self._eps(x, eps)
        coef = ops.make_coef(a, b, c, d, N, self._decoder_var_f, pairwise, x.shape[0])
        flat = self._flat_params()
        loss, z, grads = ops.elbo_fwd_bwd(self._shape, coef, flat, x, u, eps, self._ws, z_out=z_out)
        optimizer.step_flat(flat, grads)
        return loss[0], z

    def direct_steps(self, optimizer, xs, us, a, b, c, d, N, pairwise, eps=None, z_out=None, coefs=None):
        """`direct_step` over the batches xs (n, B, data_dim) [us (n, B, aux_dim)] with ONE library call
        (`ivae_elbo_adam_steps`): same kernels, same update, constant learning rate over the call; the noise of all n steps
        is one torch.randn draw.  Loss weights: (a, b, c, d, N, pairwise) for every step, or `coefs` = one such tuple per
        step (the per-iteration schedule of `iVAE.anneal`).  Returns (losses (n,), z (n, B, latent_dim))."""
        if eps is None:
            eps = torch.randn(xs.shape[0], xs.shape[1], self._shape.latent_dim, dtype=torch.float32, device=xs.device)
        if coefs is None:
            coef = ops.make_coef(a, b, c, d, N, self._decoder_var_f, pairwise, xs.shape[1])
        else:
            coef = [ops.make_coef(a_, b_, c_, d_, N_, self._decoder_var_f, pw_, xs.shape[1]) for a_, b_, c_, d_, N_, pw_ in coefs]
        flat = self._flat_params()
        m, v, taken, group = optimizer.flat_state(flat)
        b1, b2 = group['betas']
        loss, z = ops.elbo_adam_steps(self._shape, coef, flat, m, v, xs, us, eps, self._ws, taken, group['lr'], b1, b2,
                                      group['eps'], z_out=z_out)
        optimizer.advance(xs.shape[0])
        return loss[:, 0], z

    def _loss(self, x, u, a, b, c, d, N, pairwise, eps=None):
        if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (x, u)):
            # the reference's autograd would hand back dLoss/dx; the kernels form parameter gradients only -- say so
            # instead of leaving x.grad silently empty
            raise NotImplementedError('the fused path does not differentiate with respect to its inputs (x, u): detach them')
        eps = self._eps(x, eps)
        coef = ops.make_coef(a, b, c, d, N, self._decoder_var_f, pairwise, x.shape[0])
        return _ElboFn.apply(self, coef, x, u, eps, *self.parameters())


class cleanIVAE(_FusedModel):
    """nets.py:124-185."""

    def __init__(self, data_dim, latent_dim, aux_dim, n_layers=3, activation='xtanh', hidden_dim=50, slope=.1):
        super().__init__()
        self.data_dim = data_dim
        self.latent_dim = latent_dim
        self.aux_dim = aux_dim
        self.hidden_dim = hidden_dim
        self.n_layers = n_layers
        self.activation = activation
        self.slope = slope
        self.prior_mean = torch.zeros(1)
        self.logl = MLP(aux_dim, latent_dim, hidden_dim, n_layers, activation=activation, slope=slope)
        self.f = MLP(latent_dim, data_dim, hidden_dim, n_layers, activation=activation, slope=slope)
        self.decoder_var = .1 * torch.ones(1)
        self._decoder_var_f = float(self.decoder_var)
        self.g = MLP(data_dim + aux_dim, latent_dim, hidden_dim, n_layers, activation=activation, slope=slope)
        self.logv = MLP(data_dim + aux_dim, latent_dim, hidden_dim, n_layers, activation=activation, slope=slope)
        self._finish_init(data_dim, latent_dim, aux_dim, hidden_dim, n_layers, activation, slope)

    def forward(self, x, u, eps=None):
        """-> (f, g, v, s, l), nets.py:165-170."""
        f, g, v, z, l = self._forward_tensors(x, u, eps)
        return f, g, v, z, l

    def elbo(self, x, u, N, a=1., b=1., c=1., d=1., eps=None):
        """-> (loss, z): the NEGATIVE elbo, nets.py:172-185."""
        return self._loss(x, u, a, b, c, d, N, True, eps)


class cleanVAE(_FusedModel):
    """nets.py:188-243 (beta-VAE / beta-TCVAE baselines via a,b,c,d)."""

    def __init__(self, data_dim, latent_dim, n_layers=3, activation='xtanh', hidden_dim=50, slope=.1):
        super().__init__()
        self.data_dim = data_dim
        self.latent_dim = latent_dim
        self.hidden_dim = hidden_dim
        self.n_layers = n_layers
        self.activation = activation
        self.slope = slope
        self.prior_mean = torch.zeros(1)
        self.prior_var = torch.ones(1)
        self.f = MLP(latent_dim, data_dim, hidden_dim, n_layers, activation=activation, slope=slope)
        self.decoder_var = .1 * torch.ones(1)
        self._decoder_var_f = float(self.decoder_var)
        self.g = MLP(data_dim, latent_dim, hidden_dim, n_layers, activation=activation, slope=slope)
        self.logv = MLP(data_dim, latent_dim, hidden_dim, n_layers, activation=activation, slope=slope)
        self._finish_init(data_dim, latent_dim, 0, hidden_dim, n_layers, activation, slope)

    def forward(self, x, eps=None):
        """-> (f, g, v, s), nets.py:224-228."""
        f, g, v, z, _ = self._forward_tensors(x, None, eps)
        return f, g, v, z

    def elbo(self, x, u, N, a=1., b=1., c=1., d=1., eps=None):
        """-> (loss, z), nets.py:230-243 (``u`` is accepted and ignored, as there)."""
        return self._loss(x, None, a, b, c, d, N, True, eps)


class iVAE(_FusedModel):
    """nets.py:391-486."""

    def __init__(self, latent_dim, data_dim, aux_dim, prior=None, decoder=None, encoder=None,
                 n_layers=3, hidden_dim=50, activation='lrelu', slope=.1, device='cpu', anneal=False):
        super().__init__()
        self.data_dim = data_dim
        self.latent_dim = latent_dim
        self.aux_dim = aux_dim
        self.hidden_dim = hidden_dim
        self.n_layers = n_layers
        self.activation = activation
        self.slope = slope
        self.anneal_params = anneal
        for dist in (prior, decoder, encoder):
            if dist is not None and getattr(dist, 'name', None) != 'gauss':
                raise NotImplementedError('the fused iVAE path implements Gaussian prior/encoder/decoder only')
        self.prior_dist = prior if prior is not None else Normal(device=device)
        self.decoder_dist = decoder if decoder is not None else Normal(device=device)
        self.encoder_dist = encoder if encoder is not None else Normal(device=device)
        self.prior_mean = torch.zeros(1).to(device)
        self.logl = MLP(aux_dim, latent_dim, hidden_dim, n_layers, activation=activation, slope=slope, device=device)
        self.f = MLP(latent_dim, data_dim, hidden_dim, n_layers, activation=activation, slope=slope, device=device)
        self.decoder_var = .01 * torch.ones(1).to(device)
        self._decoder_var_f = float(.01 * torch.ones(1))
        self.g = MLP(data_dim + aux_dim, latent_dim, hidden_dim, n_layers, activation=activation, slope=slope,
                     device=device)
        self.logv = MLP(data_dim + aux_dim, latent_dim, hidden_dim, n_layers, activation=activation, slope=slope,
                        device=device)
        self.apply(weights_init)
        self._training_hyperparams = [1., 1., 1., 1., 1]
        self._finish_init(data_dim, latent_dim, aux_dim, hidden_dim, n_layers, activation, slope)

    def forward(self, x, u, eps=None):
        """-> (f, var), (g, v), z, (prior_mean, l); nets.py:450-455."""
        f, g, v, z, l = self._forward_tensors(x, u, eps)
        return (f, self.decoder_var), (g, v), z, (self.prior_mean, l)

    def elbo(self, x, u, eps=None):
        """-> (elbo, z): the POSITIVE elbo, nets.py:457-475."""
        if self.anneal_params:
            a, b, c, d, N = self._training_hyperparams
            loss, z = self._loss(x, u, a, b, c, d, N, True, eps)
        else:
            loss, z = self._loss(x, u, 1., 1., 1., 1., 1., False, eps)
        return loss.neg(), z

    def anneal(self, N, max_iter, it):
        """nets.py:477-486."""
        thr = int(max_iter / 1.6)
        a = 0.5 / self._decoder_var_f
        self._training_hyperparams[-1] = N
        self._training_hyperparams[0] = min(2 * a, a + a * it / thr)
        self._training_hyperparams[1] = max(1, a * .3 * (1 - it / thr))
        self._training_hyperparams[2] = min(1, it / thr)
        self._training_hyperparams[3] = max(1, a * .5 * (1 - it / thr))
        if it > thr:
            self.anneal_params = False


class VAE(_FusedModel):
    """nets.py:548-599."""

    def __init__(self, latent_dim, data_dim, decoder=None, encoder=None,
                 n_layers=3, hidden_dim=50, activation='lrelu', slope=.1, device='cpu'):
        super().__init__()
        self.data_dim = data_dim
        self.latent_dim = latent_dim
        self.hidden_dim = hidden_dim
        self.n_layers = n_layers
        self.activation = activation
        self.slope = slope
        for dist in (decoder, encoder):
            if dist is not None and getattr(dist, 'name', None) != 'gauss':
                raise NotImplementedError('the fused VAE path implements Gaussian encoder/decoder only')
        self.decoder_dist = decoder if decoder is not None else Normal(device=device)
        self.encoder_dist = encoder if encoder is not None else Normal(device=device)
        self.prior_dist = Normal(device)
        self.prior_mean = torch.zeros(1).to(device)
        self.prior_var = torch.ones(1).to(device)
        self.f = MLP(latent_dim, data_dim, hidden_dim, n_layers, activation=activation, slope=slope, device=device)
        self.decoder_var = .01 * torch.ones(1).to(device)
        self._decoder_var_f = float(.01 * torch.ones(1))
        self.g = MLP(data_dim, latent_dim, hidden_dim, n_layers, activation=activation, slope=slope, device=device)
        self.logv = MLP(data_dim, latent_dim, hidden_dim, n_layers, activation=activation, slope=slope, device=device)
        self._finish_init(data_dim, latent_dim, 0, hidden_dim, n_layers, activation, slope)

    def forward(self, x, eps=None):
        """-> (f, var), (g, v), z, (prior_mean, prior_var); nets.py:587-591."""
        f, g, v, z, _ = self._forward_tensors(x, None, eps)
        return (f, self.decoder_var), (g, v), z, (self.prior_mean, self.prior_var)

    def elbo(self, x, eps=None):
        """-> (elbo, z), nets.py:593-599."""
        loss, z = self._loss(x, None, 1., 1., 1., 1., 1., False, eps)
        return loss.neg(), z
