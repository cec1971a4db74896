"""Autograd functions and modules on the operators of ``gact.fused``.

    layers.convert(model)                      nn.LayerNorm / nn.Linear (and the activation behind a Linear in nn.Sequential)
    y = layers.linear(x, w, b, activation="gelu", residual=r)
    y = layers.layer_norm(x, w, b, eps)

What such a layer keeps for its backward pass is its own 8-bit checkpoint (or, at level L0 / with
``config.compress_activation`` off, the tensors themselves); a ``Controller``'s hooks see int8 codes and parameters, leave
both alone and go on compressing everything else the model saves.  Converted layers therefore have a fixed width of 8 bits:
auto precision adapts the other tensors.  ``config.stochastic_checkpoints`` rounds the codes stochastically instead of to
nearest.

Linear layers compute in float16 / bfloat16 (under autocast input and parameters are cast to its type, as torch does); layer norm
keeps the type of its input (torch's returns float32 under autocast).
"""
import math

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from gact import fused
from gact.conf import config
from gact.fused import Checkpoint8, LayerNormSaved, LinearSaved

_calls = 0


def _next_seed(device=None):
    """None (round to nearest), or a seed of its own for every call: from torch's seed, the rank and a running number.  While the
    device's stream is captured it is drawn on the device by torch's generator, whose state moves on from replay to replay."""
    if not config.stochastic_checkpoints:
        return None
    global _calls
    _calls += 1
    rank = torch.distributed.get_rank() if torch.distributed.is_available() and torch.distributed.is_initialized() else 0
    if device is not None and torch.cuda.is_current_stream_capturing():
        seed = torch.empty(1, dtype=torch.int64, device=device).random_()
        return seed.add_(rank << 40) if rank else seed
    return (torch.initial_seed() * 0x9E3779B97F4A7C15 + (rank << 40) + 2 * _calls) & 0xFFFFFFFFFFFFFFFF


def _keeps_graph(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _flat(kept):
    """(tensor, shape, dtype) of a Checkpoint8 or a tensor (shape None), for save_for_backward."""
    if type(kept) is Checkpoint8:
        return kept.buf, kept.shape, kept.dtype
    return kept, None, None


def _unflat(t, shape, dtype):
    return t if shape is None else Checkpoint8(t, shape, dtype)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, compress, seed):
        y, s = fused.op_layer_norm(x, weight, bias, eps, compress=compress, seed=seed, center=True)
        t, *ctx.kept = _flat(s.x)
        ctx.save_for_backward(t, s.stats, s.weight)
        ctx.meta = (s.shape, s.dtype, s.param_dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        t, stats, weight = ctx.saved_tensors
        saved = LayerNormSaved(_unflat(t, *ctx.kept), stats, weight, *ctx.meta)
        n = ctx.needs_input_grad
        return (*fused.op_layer_norm_backward(dy, saved, (n[0], n[1], n[2])), None, None, None)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, compress, seed, given, keep_input):
        # Under autocast the parameters are cast here and again in backward.  What is saved is the weight itself, detached: saved-tensor
        # hooks take a tensor that requires a gradient and is no parameter they know (a cast copy, a computed weight) for an activation,
        # and would quantize it.
        w, b = _autocast(weight, bias)
        # Only what a gradient will need: the input for the weight's, the weight for the input's, the pre-activation for any of the three.
        n = ctx.needs_input_grad
        if not (n[0] or n[1] or n[2]):
            return fused.op_linear(x, w, b, activation, residual, save=False)[0]
        keep_input = keep_input or n[1]
        ck = None if given is None or not keep_input else Checkpoint8(given, x.shape, x.dtype)
        y, s = fused.op_linear(x, w, b, activation, residual, compress=compress, seed=seed, checkpoint=ck, keep_input=keep_input)
        xt, *ctx.x = _flat(s.x)
        zt, *ctx.z = _flat(s.z)
        ctx.save_for_backward(xt, zt, weight.detach() if n[0] else None)
        ctx.meta = (activation, s.out_shape, s.has_bias, s.in_features)
        ctx.param_dtypes = weight.dtype, None if bias is None else bias.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        n = ctx.needs_input_grad
        if not (n[0] or n[1] or n[2]):
            return (None,) * 3 + (dy,) + (None,) * 5
        xt, zt, weight = ctx.saved_tensors
        saved = LinearSaved(_unflat(xt, *ctx.x), _unflat(zt, *ctx.z), None if weight is None else weight.to(dy.dtype), *ctx.meta)
        dx, dw, db = fused.op_linear_backward(dy, saved, (n[0], n[1], n[2]))
        wt, bt = ctx.param_dtypes
        return dx, None if dw is None else dw.to(wt), None if db is None else db.to(bt), (dy if n[3] else None), None, None, None, None, None


def layer_norm(input, weight=None, bias=None, eps=1e-5, compress=None):
    """Layer norm over the last dimension, differentiable; what it keeps is decided by ``compress`` (None: by the level,
    ``config.compress_activation``): the checkpoint of the input minus its row's mean, or the input itself.  Parameters are of
    the input's type or float32; under autocast others (bfloat16 ones with a float32 input, say) are widened to float32."""
    params = [p for p in (weight, bias) if p is not None]
    if torch.is_autocast_enabled("cuda") and any(p.dtype not in (input.dtype, torch.float32) or p.dtype != params[0].dtype for p in params):
        weight, bias = (p if p is None or p.dtype == torch.float64 else p.float() for p in (weight, bias))
    if not _keeps_graph(input, weight, bias):
        return fused.op_layer_norm(input, weight, bias, eps, save=False)[0]
    compress = config.compress_activation if compress is None else compress
    return _LayerNorm.apply(input, weight, bias, eps, compress, _next_seed(input.device) if compress else None)


def _autocast_dtype(t):
    """The type that a linear layer computes a tensor in."""
    if not torch.is_autocast_enabled("cuda") or not t.is_floating_point() or t.dtype == torch.float64:
        return t.dtype
    return torch.get_autocast_dtype("cuda")


def _autocast(*tensors):
    return tuple(t if t is None else t.to(_autocast_dtype(t)) for t in tensors)


def linear(input, weight, bias=None, activation=None, residual=None, compress=None, checkpoint=None, keep_input=None):
    """activation(input W^T + bias) + residual, differentiable; see ``gact.fused.op_linear``.  ``compress`` as in
    ``layer_norm``; ``checkpoint``: a Checkpoint8 of the input (in the type it is computed in) to share.  ``keep_input``: whether the
    input is kept although the weight asks for no gradient; None: not for a frozen parameter, but for a plain tensor (whose
    ``grad_fn.saved_tensors`` then hold it).  A residual of another type is an error, but under autocast it is added to the
    result as torch adds it, in the wider of the two types."""
    input, = _autocast(input)
    if input.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError("gact.layers.linear computes in float16 or bfloat16: cast the model or use torch.autocast "
                           "(got an input of %s)" % input.dtype)
    if residual is not None and residual.dtype != input.dtype and torch.is_autocast_enabled("cuda"):
        # as torch's sum: the wider type (an fp32 residual stream keeps its bits)
        y = linear(input, weight, bias, activation, None, compress, checkpoint, keep_input)
        if residual.shape != y.shape:
            raise ValueError("residual must have shape %s, got %s" % (tuple(y.shape), tuple(residual.shape)))
        return y + residual
    if not _keeps_graph(input, weight, bias, residual):
        return fused.op_linear(input, *_autocast(weight, bias), activation, residual, save=False)[0]
    compress = config.compress_activation if compress is None else compress
    given = None
    if compress and checkpoint is not None:
        if checkpoint.shape != input.shape or checkpoint.dtype != input.dtype:
            raise ValueError("checkpoint is of a %s tensor of shape %s" % (checkpoint.dtype, tuple(checkpoint.shape)))
        given = checkpoint.buf
    return _Linear.apply(input, weight, bias, residual, activation, compress, _next_seed(input.device) if compress else None, given,
                         not isinstance(weight, nn.Parameter) if keep_input is None else keep_input)


class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm that keeps its input in 8 bits."""

    def forward(self, input):
        shape = tuple(self.normalized_shape)
        if input.shape[-len(shape):] != shape:
            raise RuntimeError("normalized_shape %s does not fit an input of shape %s" % (shape, tuple(input.shape)))
        if len(shape) == 1:
            return layer_norm(input, self.weight, self.bias, self.eps)
        x = input.flatten(-len(shape))
        w = None if self.weight is None else self.weight.flatten()
        b = None if self.bias is None else self.bias.flatten()
        return layer_norm(x, w, b, self.eps).view(input.shape)


class Linear(nn.Linear):
    """nn.Linear with the activation behind it in its epilogue; keeps its input and pre-activation in 8 bits."""

    def __init__(self, in_features, out_features, bias=True, activation=None, device=None, dtype=None):
        super().__init__(in_features, out_features, bias, device, dtype)
        self.activation = activation
        self._shared = None

    def forward(self, input, residual=None):
        shared, self._shared = self._shared, None
        checkpoint = None
        # It was made in the type that the parent was called under (a forward pass that enters autocast by itself computes in
        # another) and on its stream (a layer on another one could read it before it is there, and outlive it).
        if shared is not None and shared[1] is input and shared[2] == input._version and shared[0].dtype == _autocast_dtype(input) \
                and shared[3] == _stream(input):
            checkpoint = shared[0]
        return linear(input, self.weight, self.bias, self.activation, residual, checkpoint=checkpoint)

    def extra_repr(self):
        return super().extra_repr() + ("" if self.activation is None else ", activation=%s" % self.activation)


def _stream(x):
    return torch.cuda.current_stream(x.device) if x.is_cuda else None


class _SharedInput:
    """The hooks of ``share_input``: an object whose methods they are, so that a copied or pickled parent has its own, with its own
    layers."""

    def __init__(self, children):
        self.children = list(children)

    def before(self, module, args):
        x = args[0] if args else None
        # (frozen weights keep no input)
        if isinstance(x, torch.Tensor) and config.compress_activation and _keeps_graph(*(c.weight for c in self.children)):
            cast = _autocast(x)[0]
            if cast.dtype in (torch.float16, torch.bfloat16):
                ck = fused.op_checkpoint8(cast.detach(), _next_seed(x.device))
                for c in self.children:
                    c._shared = (ck, x, x._version, _stream(x))

    def after(self, module, args, output):
        for c in self.children:
            c._shared = None


def share_input(parent, children):
    """Lets linear layers that ``parent`` calls with its own first argument share one checkpoint of it (the query, key and
    value layers of an attention block): made when ``parent`` is called, used by the next call of each child that is given
    that very tensor, unmodified, on the same stream, and dropped when ``parent`` returns."""
    shared = _SharedInput(children)
    parent.register_forward_pre_hook(shared.before)
    parent.register_forward_hook(shared.after, always_call=True)


def activation_name(module):
    """The name ``linear`` knows an activation module by, or None."""
    if type(module) is nn.GELU:
        return "gelu_tanh" if module.approximate == "tanh" else "gelu"
    return {nn.ReLU: "relu", nn.SiLU: "silu"}.get(type(module))


def _as_linear(m, activation=None):
    out = Linear.__new__(Linear)
    nn.Module.__init__(out)
    out.in_features, out.out_features, out.weight, out.bias = m.in_features, m.out_features, m.weight, m.bias
    out.activation, out._shared = activation, None
    out.train(m.training)
    return out


def _as_layer_norm(m):
    out = LayerNorm.__new__(LayerNorm)
    nn.Module.__init__(out)
    out.normalized_shape, out.eps, out.elementwise_affine = m.normalized_shape, m.eps, m.elementwise_affine
    out.weight, out.bias = m.weight, m.bias
    out.train(m.training)
    return out


def convert(module):
    """Replaces, in place, every nn.LayerNorm and nn.Linear under ``module`` by the layers above, which take over the very
    parameters; a GELU / ReLU / SiLU that follows a Linear inside an nn.Sequential moves into its epilogue.  Subclasses of
    nn.Linear / nn.LayerNorm, layers that carry hooks, layers in float64 and norms over more elements than the operator takes (16384) stay as
    they are.  Returns ``module`` (or its replacement)."""
    if _hooked(module) or any(p.dtype == torch.float64 for p in module._parameters.values() if p is not None):
        pass
    elif type(module) is nn.Linear:
        return _as_linear(module)
    elif type(module) is nn.LayerNorm and math.prod(module.normalized_shape) <= fused.LAYER_NORM_MAX_COLS:
        return _as_layer_norm(module)
    names = list(module._modules)
    for i, name in enumerate(names):
        child = module._modules[name]
        if child is None:
            continue
        new = convert(child)
        # (a layer that was one of these before may be used, or watched by hooks, elsewhere too: it keeps its output)
        if type(module) is nn.Sequential and new is not child and type(new) is Linear and i + 1 < len(names):
            act = activation_name(module._modules[names[i + 1]])
            if act is not None and not _hooked(module._modules[names[i + 1]]):
                new.activation = act
                module._modules[names[i + 1]] = nn.Identity()
        module._modules[name] = new
    return module


def _hooked(m):
    return bool(m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks)
