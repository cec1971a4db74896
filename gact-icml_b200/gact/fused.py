"""Training operators that keep their own activations as 8-bit checkpoints and whose backward passes work from them.

    c = op_checkpoint8(x)                         8-bit codes, one power-of-two scale per 32 elements of a row
    x = op_restore8(c)
    y, saved = op_layer_norm(x, weight, bias)     layer norm over the last dimension
    dx, dw, db = op_layer_norm_backward(dy, saved)
    y, saved = op_linear(x, weight, bias, activation="gelu", residual=r)      act(x W^T + b) + r
    dx, dw, db = op_linear_backward(dy, saved)

The compression of saved tensors (``gact.ops``) restores a tensor in full before a library kernel reads it; these
operators read the codes themselves.  ``gact.layers`` wraps them for autograd.  Like ``gact.ops``, nothing here falls
back to another implementation, and kernels run on the current stream of the tensors' device.

Products and layer norm's rings wait for their copies with a limit.  A wait that runs out leaves results incomplete, and the next
call of any operator here that finds it has happened raises RuntimeError; ``check()`` waits for the device and raises for
everything up to then (after the last step of a run, say).
"""
import torch

from gact import _native as nv

try:
    from gact import _fused
except ImportError as e:
    raise ImportError("gact/_fused.so is missing or does not load (%s): build it with `python gact-icml_b200/build.py`.  "
                      "gact has no fallback path." % e)

LAYER_NORM_MAX_COLS = 16384


def check():
    """Waits for the current device and raises RuntimeError if a wait of an operator's copies has run out there since the last check
    (one that a call has raised for already among them)."""
    torch.cuda.synchronize()
    nv.check_pipeline("gact.fused")


# ---------------------------------------------------------------------------------------------------------------
# checkpoints
# ---------------------------------------------------------------------------------------------------------------
class Checkpoint8:
    """A tensor kept in 8 bits: ``buf`` (int8, one dimension) holds the codes and behind them the scales, ``shape`` and
    ``dtype`` say what it restores to.  ``codes``: int8 (rows, pitch), pitch = last dimension rounded up to 32; ``scales``: int8
    (rows, pitch / 32), the bits of an unsigned biased exponent."""
    __slots__ = ("buf", "shape", "dtype")

    def __init__(self, buf, shape, dtype):
        self.buf, self.shape, self.dtype = buf, shape, dtype

    def _layout(self):
        rows = 1
        for n in self.shape[:-1]:
            rows *= n
        return rows, (self.shape[-1] + nv.BLOCK8 - 1) // nv.BLOCK8 * nv.BLOCK8

    @property
    def codes(self):
        rows, pitch = self._layout()
        return self.buf[:rows * pitch].view(rows, pitch)

    @property
    def scales(self):
        rows, pitch = self._layout()
        return self.buf[rows * pitch:].view(rows, pitch // nv.BLOCK8)

    @property
    def nbytes(self):
        return self.buf.numel()


def _unwrap(kept):
    return kept.buf if type(kept) is Checkpoint8 else kept


def op_checkpoint8(input, seed=None):
    """8-bit checkpoint of a float32 / float16 / bfloat16 tensor, blocks of 32 along its last dimension.

    Rounds to nearest, or with a ``seed`` stochastically (unbiased; the same seed gives the same codes).  A seed is a number, or
    an int64 tensor of one element on the input's device, which the kernel reads: in a captured graph a number is repeated by
    every replay, a tensor's value is that of the replay.  A block that holds a NaN or an infinity restores to NaN throughout."""
    return Checkpoint8(_fused.checkpoint8(input, seed), input.shape, input.dtype)


def op_restore8(c, dtype=None):
    """The tensor a checkpoint stands for, in its own type or in ``dtype``."""
    if type(c) is not Checkpoint8:
        raise TypeError("op_restore8 takes a Checkpoint8")
    return _fused.restore8(c.buf, tuple(c.shape), c.dtype if dtype is None else dtype)


# ---------------------------------------------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------------------------------------------
class LayerNormSaved:
    """What layer norm's backward pass needs: the input (a Checkpoint8 of it or of its deviation from the rows' means, or the
    tensor itself), per row what is still to be taken off (the mean, or 0) and 1 / deviation (fp32 (rows, 2)), and the weight."""
    __slots__ = ("x", "stats", "weight", "shape", "dtype", "param_dtype")

    def __init__(self, x, stats, weight, shape, dtype, param_dtype):
        self.x, self.stats, self.weight = x, stats, weight
        self.shape, self.dtype, self.param_dtype = shape, dtype, param_dtype


def op_layer_norm(input, weight=None, bias=None, eps=1e-5, compress=True, seed=None, save=True, center=False):
    """(y, saved): layer norm over the last dimension (at most 16384) of a float32 / float16 / bfloat16 tensor.

    weight, bias: of the input's type or float32, or None.  ``compress``: keep the input as a Checkpoint8 (made in the same
    pass; with a ``seed`` rounded stochastically) for the backward pass, else the input itself.  ``save`` False: forward
    only, saved is None.  ``center``: the checkpoint is that of the input minus its row's mean, and its error stays below 1/127
    of the row's largest deviation.  Codes of the input itself (which other operators can share) have a step of 1/127 to
    1/64 of the largest magnitude of 32 neighbours, mean included: where a row's mean is large against its deviation they
    leave the gradients little to work from."""
    y, kept, stats, w = _fused.layer_norm(input, weight, bias, eps, compress, seed, save, center)
    if not save:
        return y, None
    param = weight if weight is not None else bias
    if compress:
        kept = Checkpoint8(kept, input.shape, torch.float32 if center else input.dtype)
    return y, LayerNormSaved(kept, stats, w, input.shape, input.dtype, input.dtype if param is None else param.dtype)


def op_layer_norm_backward(grad_output, saved, needs=(True, True, True)):
    """(grad of the input, of weight, of bias) from what op_layer_norm saved; None where ``needs`` says so."""
    if grad_output.shape != saved.shape:
        raise ValueError("grad_output must have shape %s, got %s" % (tuple(saved.shape), tuple(grad_output.shape)))
    if grad_output.dtype != saved.dtype:
        raise RuntimeError("The type of grad_output is not correct!")
    return _fused.layer_norm_backward(grad_output, _unwrap(saved.x), saved.stats, saved.weight, saved.param_dtype == torch.float32, *needs)


# ---------------------------------------------------------------------------------------------------------------
# linear
# ---------------------------------------------------------------------------------------------------------------
class LinearSaved:
    """What the backward pass of a linear layer needs: its input (for the weight's gradient) and, with an activation, its
    pre-activation, each a Checkpoint8 or a tensor, and the weight (for the input's gradient; without it ``in_features``)."""
    __slots__ = ("x", "z", "weight", "activation", "out_shape", "has_bias", "in_features")

    def __init__(self, x, z, weight, activation, out_shape, has_bias, in_features=None):
        self.x, self.z, self.weight, self.activation, self.out_shape, self.has_bias = x, z, weight, activation, out_shape, has_bias
        self.in_features = weight.shape[-1] if in_features is None else in_features


def op_linear(input, weight, bias=None, activation=None, residual=None, compress=True, seed=None, save=True, checkpoint=None, keep_input=True):
    """(y, saved): y = activation(input W^T + bias) + residual for float16 / bfloat16 tensors, fp32 accumulation.

    activation: None, "relu", "gelu" (erf), "gelu_tanh" or "silu".  ``compress``: keep input and pre-activation as
    Checkpoint8 for the backward pass (with a ``seed`` rounded stochastically), else as tensors.  ``checkpoint``: a
    Checkpoint8 of this very input that is already there (several layers reading one tensor share it).  ``save`` False:
    forward only, saved is None; ``keep_input`` False: a frozen weight, whose gradient nobody will ask for, keeps no input."""
    act = nv.ACT_CODE.get(activation)
    if act is None:
        raise ValueError("unknown activation %r" % (activation,))
    given = None
    if checkpoint is not None:
        if type(checkpoint) is not Checkpoint8:
            raise TypeError("checkpoint must be a Checkpoint8")
        if checkpoint.shape != input.shape or checkpoint.dtype != input.dtype:
            raise ValueError("checkpoint is of a %s tensor of shape %s" % (checkpoint.dtype, tuple(checkpoint.shape)))
        given = checkpoint.buf
    y, kept, z = _fused.linear(input, weight, bias, act, residual, compress, seed, save, given, keep_input)
    if not save:
        return y, None
    if compress:
        if kept is not None:
            kept = checkpoint if checkpoint is not None else Checkpoint8(kept, input.shape, input.dtype)
        if z is not None:
            z = Checkpoint8(z, y.shape, input.dtype)
    return y, LinearSaved(kept, z, weight, activation, y.shape, bias is not None)


def op_linear_backward(grad_output, saved, needs=(True, True, True)):
    """(grad of the input, of weight, of bias) from what op_linear saved; None where ``needs`` says so or there is no bias.
    The gradient of a residual is grad_output itself."""
    if grad_output.shape != saved.out_shape:
        raise ValueError("grad_output must have shape %s, got %s" % (tuple(saved.out_shape), tuple(grad_output.shape)))
    return _fused.linear_backward(grad_output, saved.weight, nv.ACT_CODE[saved.activation], _unwrap(saved.x), _unwrap(saved.z), needs[0], needs[1],
                                  needs[2] and saved.has_bias, saved.in_features)
