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
"""
import torch

from gact import _native as nv
from gact import ops as _ops

_LIB = nv.lib
_HALF = (torch.float16, torch.bfloat16)
LAYER_NORM_MAX_COLS = 16384


def _count(n):
    _ops.launch_count += n


def _seed(seed):
    """(stochastic flag, 64-bit seed) of a `seed` argument: None rounds to nearest."""
    return (0, 0) if seed is None else (1, int(seed) & 0xFFFFFFFFFFFFFFFF)


def _check_tensor(t, name, dtypes=None, like=None):
    nv.require_cuda(t, name)
    if t.layout != torch.strided:
        raise RuntimeError("%s must be a dense tensor" % name)
    if dtypes is not None and t.dtype not in dtypes:
        raise RuntimeError("The type of %s is not correct!" % name)
    if like is not None and t.device != like.device:
        raise RuntimeError("%s is on %s, the input on %s" % (name, t.device, like.device))


def _rows(t, cols):
    """(tensor, rows, pitch in elements) of t as rows of `cols` elements with unit stride inside a row; copies only what
    cannot be described that way."""
    if t.dim() != 2:
        t = t.reshape(-1, cols) if t.numel() else t.reshape(_ops._numel(t.shape[:-1]), cols)
    rows = t.shape[0]
    if cols > 1 and t.stride(1) != 1:
        t = t.contiguous()
    ld = t.stride(0) if rows > 1 else cols
    if ld < cols:                                   # expanded rows
        t = t.contiguous()
        ld = cols
    return t, rows, ld


def _operand(t, rows, cols, ld, stream):
    """(tensor to keep alive, address, pitch) of a matrix that a tensor map can describe: base and pitch multiples of 16
    bytes.  Anything else is copied to such a pitch first."""
    ptr = t.data_ptr()
    if ld % 8 == 0 and ptr % 16 == 0:
        return t, ptr, ld
    pitch = (cols + 7) // 8 * 8
    out = torch.empty((rows, pitch), dtype=t.dtype, device=t.device)
    nv.check(_LIB.gact_repitch16(ptr, ld, rows, cols, out.data_ptr(), pitch, stream), "gact_repitch16")
    _count(1)
    return out, out.data_ptr(), pitch


def _scratch(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _ptr(t):
    return None if t is None else t.data_ptr()


# ---------------------------------------------------------------------------------------------------------------
# checkpoints
# ---------------------------------------------------------------------------------------------------------------
class Checkpoint8:
    """A tensor kept in 8 bits: ``codes`` int8 (rows, pitch), ``scales`` int8 (rows, pitch / 32; the bits of an unsigned
    biased exponent), and the ``shape`` and ``dtype`` it restores to.  pitch = last dimension rounded up to 32."""
    __slots__ = ("codes", "scales", "shape", "dtype")

    def __init__(self, codes, scales, shape, dtype):
        self.codes, self.scales, self.shape, self.dtype = codes, scales, shape, dtype

    @property
    def nbytes(self):
        return self.codes.numel() + self.scales.numel()


def _empty_checkpoint(rows, cols, shape, dtype, device):
    pitch = (cols + nv.BLOCK8 - 1) // nv.BLOCK8 * nv.BLOCK8
    # one allocation: codes, then scales
    buf = torch.empty(rows * pitch + rows * (pitch // nv.BLOCK8), dtype=torch.int8, device=device)
    n = rows * pitch
    return Checkpoint8(buf[:n].view(rows, pitch), buf[n:].view(rows, pitch // nv.BLOCK8), shape, dtype)


def op_checkpoint8(input, seed=None):
    """8-bit checkpoint of a float32 / float16 / bfloat16 tensor, blocks of 32 along its last dimension.

    Rounds to nearest, or with a ``seed`` stochastically (unbiased; the same seed gives the same codes).  A block that
    holds a NaN or an infinity restores to NaN throughout."""
    _check_tensor(input, "input", nv.DTYPE_CODE)
    if input.dim() == 0:
        raise ValueError("input needs at least one dimension")
    cols = input.shape[-1]
    shape, dtype = input.shape, input.dtype
    if input.numel() == 0:
        return _empty_checkpoint(_ops._numel(shape[:-1]), cols, shape, dtype, input.device)
    x, rows, ld = _rows(input, cols)
    c = _empty_checkpoint(rows, cols, shape, dtype, x.device)
    stoch, s = _seed(seed)
    guard, stream = nv.guard_and_stream(x)
    with guard:
        nv.check(_LIB.gact_checkpoint8(x.data_ptr(), nv.DTYPE_CODE[dtype], rows, cols, ld, stoch, s, c.codes.data_ptr(), c.scales.data_ptr(),
                                       stream), "gact_checkpoint8")
    _count(1)
    return c


def _check_checkpoint(c, cols, rows, like, name):
    if not isinstance(c, Checkpoint8):
        raise TypeError("%s must be a Checkpoint8" % name)
    pitch = (cols + nv.BLOCK8 - 1) // nv.BLOCK8 * nv.BLOCK8
    for t, shape, what in ((c.codes, (rows, pitch), "codes"), (c.scales, (rows, pitch // nv.BLOCK8), "scales")):
        nv.require_cuda(t, "%s.%s" % (name, what))
        if tuple(t.shape) != shape or not t.is_contiguous() or t.element_size() != 1:
            raise ValueError("%s.%s must be contiguous bytes of shape %s" % (name, what, shape))
        if like is not None and t.device != like.device:
            raise RuntimeError("%s is on %s, the input on %s" % (name, t.device, like.device))


def op_restore8(c, dtype=None):
    """The tensor a checkpoint stands for, in its own type or in ``dtype``."""
    if not isinstance(c, Checkpoint8):
        raise TypeError("op_restore8 takes a Checkpoint8")
    dtype = c.dtype if dtype is None else dtype
    if dtype not in nv.DTYPE_CODE:
        raise RuntimeError("The type of the result is not correct!")
    shape = tuple(c.shape)
    cols, rows = shape[-1], _ops._numel(shape[:-1])
    _check_checkpoint(c, cols, rows, None, "checkpoint")
    if c.scales.device != c.codes.device:
        raise RuntimeError("codes and scales are on different devices")
    out = torch.empty(shape, dtype=dtype, device=c.codes.device)
    if out.numel() == 0:
        return out
    guard, stream = nv.guard_and_stream(out)
    with guard:
        nv.check(_LIB.gact_restore8(c.codes.data_ptr(), c.scales.data_ptr(), rows, cols, nv.DTYPE_CODE[dtype], out.data_ptr(), cols, stream),
                 "gact_restore8")
    _count(1)
    return out


# ---------------------------------------------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------------------------------------------
class LayerNormSaved:
    """What layer norm's backward pass needs: the input (a Checkpoint8, or the tensor itself), the row statistics and
    the weight."""
    __slots__ = ("x", "mean", "rstd", "weight", "shape", "dtype", "param_dtype")

    def __init__(self, x, mean, rstd, weight, shape, dtype, param_dtype):
        self.x, self.mean, self.rstd, self.weight = x, mean, rstd, weight
        self.shape, self.dtype, self.param_dtype = shape, dtype, param_dtype


def _check_params(weight, bias, cols, like):
    """Type code of weight and bias: that of the input, or float32; both alike."""
    dt = None
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        _check_tensor(t, name, like=like)
        if tuple(t.shape) != (cols,):
            raise ValueError("%s must have shape (%d,), got %s" % (name, cols, tuple(t.shape)))
        if t.dtype not in (like.dtype, torch.float32) or (dt is not None and t.dtype != dt):
            raise RuntimeError("The type of %s is not correct!" % name)
        dt = t.dtype
    return like.dtype if dt is None else dt


def op_layer_norm(input, weight=None, bias=None, eps=1e-5, compress=True, seed=None, save=True):
    """(y, saved): layer norm over the last dimension of a float32 / float16 / bfloat16 tensor.

    weight, bias: of the input's type or float32, or None.  ``compress``: keep the input as a Checkpoint8 (made in the same
    pass) for the backward pass, else the input itself.  ``save`` False: forward only, saved is None."""
    _check_tensor(input, "input", nv.DTYPE_CODE)
    if input.dim() == 0:
        raise ValueError("input needs at least one dimension")
    cols = input.shape[-1]
    if not 1 <= cols <= LAYER_NORM_MAX_COLS:
        raise ValueError("layer norm takes rows of 1 to %d elements, got %d" % (LAYER_NORM_MAX_COLS, cols))
    pdt = _check_params(weight, bias, cols, input)
    shape, dtype = input.shape, input.dtype
    x, rows, ld = _rows(input, cols)
    w = None if weight is None else weight.contiguous()
    b = None if bias is None else bias.contiguous()
    y = torch.empty(shape, dtype=dtype, device=x.device)
    saved, c, stats = None, None, None
    if save:
        stats = torch.empty((2, rows), dtype=torch.float32, device=x.device)
        if compress:
            c = _empty_checkpoint(rows, cols, shape, dtype, x.device)
        saved = LayerNormSaved(c if compress else x, stats[0], stats[1], w, shape, dtype, pdt)
    if rows == 0:
        return y, saved
    stoch, s = _seed(seed)
    mean = None if stats is None else stats.data_ptr()
    guard, stream = nv.guard_and_stream(x)
    with guard:
        nv.check(_LIB.gact_layer_norm(x.data_ptr(), nv.DTYPE_CODE[dtype], rows, cols, ld, _ptr(w), _ptr(b), nv.DTYPE_CODE[pdt], float(eps),
                                      y.data_ptr(), mean, None if mean is None else mean + 4 * rows,
                                      None if c is None else c.codes.data_ptr(), None if c is None else c.scales.data_ptr(), stoch, s, stream),
                 "gact_layer_norm")
    _count(1)
    return y, saved


def op_layer_norm_backward(grad_output, saved, needs=(True, True, True)):
    """(grad of the input, of weight, of bias) from what op_layer_norm saved; None where ``needs`` says so."""
    cols = saved.shape[-1]
    nv.require_cuda(grad_output, "grad_output")
    _check_tensor(grad_output, "grad_output", (saved.dtype,), like=saved.mean)
    if grad_output.shape != saved.shape:
        raise ValueError("grad_output must have shape %s, got %s" % (tuple(saved.shape), tuple(grad_output.shape)))
    dy, rows, ld = _rows(grad_output, cols)
    dev = dy.device
    x, xld, c = None, 0, None
    if isinstance(saved.x, Checkpoint8):
        c = saved.x
        _check_checkpoint(c, cols, rows, dy, "saved input")
    else:
        x, _, xld = _rows(saved.x, cols)
    dx = torch.empty(saved.shape, dtype=saved.dtype, device=dev) if needs[0] else None
    dw = torch.empty(cols, dtype=saved.param_dtype, device=dev) if needs[1] else None
    db = torch.empty(cols, dtype=saved.param_dtype, device=dev) if needs[2] else None
    if not any(needs):
        return dx, dw, db
    scratch = _scratch(_LIB.gact_layer_norm_backward_scratch_bytes(rows, cols), dev) if needs[1] or needs[2] else None
    guard, stream = nv.guard_and_stream(dy)
    with guard:
        nv.check(_LIB.gact_layer_norm_backward(dy.data_ptr(), nv.DTYPE_CODE[saved.dtype], rows, cols, ld, _ptr(x), xld,
                                               None if c is None else c.codes.data_ptr(), None if c is None else c.scales.data_ptr(),
                                               saved.mean.data_ptr(), saved.rstd.data_ptr(), _ptr(saved.weight),
                                               nv.DTYPE_CODE[saved.param_dtype], _ptr(dx), _ptr(dw), _ptr(db), _ptr(scratch), stream),
                 "gact_layer_norm_backward")
    _count(1 + (scratch is not None))
    return dx, dw, db


# ---------------------------------------------------------------------------------------------------------------
# linear
# ---------------------------------------------------------------------------------------------------------------
class LinearSaved:
    """What the backward pass of a linear layer needs: its input and (with an activation) its pre-activation, each a
    Checkpoint8 or a tensor, and the weight."""
    __slots__ = ("x", "z", "weight", "activation", "in_shape", "out_shape", "dtype", "has_bias")

    def __init__(self, x, z, weight, activation, in_shape, out_shape, dtype, has_bias):
        self.x, self.z, self.weight, self.activation = x, z, weight, activation
        self.in_shape, self.out_shape, self.dtype, self.has_bias = in_shape, out_shape, dtype, has_bias


def op_linear(input, weight, bias=None, activation=None, residual=None, compress=True, seed=None, save=True, checkpoint=None):
    """(y, saved): y = activation(input W^T + bias) + residual for float16 / bfloat16 tensors, fp32 accumulation.

    activation: None, "relu", "gelu" (erf), "gelu_tanh" or "silu".  ``compress``: keep input and pre-activation as
    Checkpoint8 for the backward pass, else as tensors.  ``checkpoint``: a Checkpoint8 of this very input that is already
    there (several layers reading one tensor share it).  ``save`` False: forward only, saved is None."""
    _check_tensor(input, "input", _HALF)
    _check_tensor(weight, "weight", (input.dtype,), like=input)
    if input.dim() == 0 or weight.dim() != 2 or input.shape[-1] != weight.shape[1]:
        raise ValueError("input %s does not fit weight %s" % (tuple(input.shape), tuple(weight.shape)))
    if activation not in nv.ACT_CODE:
        raise ValueError("unknown activation %r" % (activation,))
    act = nv.ACT_CODE[activation]
    cout, cin = weight.shape
    if cin == 0 or cout == 0:
        raise ValueError("a linear layer needs at least one input and one output feature")
    shape, dtype = input.shape, input.dtype
    out_shape = shape[:-1] + (cout,)
    if bias is not None:
        _check_tensor(bias, "bias", (dtype,), like=input)
        if tuple(bias.shape) != (cout,):
            raise ValueError("bias must have shape (%d,), got %s" % (cout, tuple(bias.shape)))
        bias = bias.contiguous()
    x, rows, ld = _rows(input, cin)
    res, ld_res = None, 0
    if residual is not None:
        _check_tensor(residual, "residual", (dtype,), like=input)
        if residual.shape != out_shape:
            raise ValueError("residual must have shape %s, got %s" % (tuple(out_shape), tuple(residual.shape)))
        res, _, ld_res = _rows(residual, cout)
    if checkpoint is not None:
        _check_checkpoint(checkpoint, cin, rows, input, "checkpoint")
        if checkpoint.shape != shape or checkpoint.dtype != dtype:
            raise ValueError("checkpoint is of a %s tensor of shape %s" % (checkpoint.dtype, tuple(checkpoint.shape)))
    dev = x.device
    y = torch.empty(out_shape, dtype=dtype, device=dev)
    stoch, s = _seed(seed)
    saved, kept, z, zc = None, None, None, None
    if save:
        if act and compress:
            zc = _empty_checkpoint(rows, cout, out_shape, dtype, dev)
        elif act:
            z = torch.empty((rows, cout), dtype=dtype, device=dev)
        kept = (checkpoint if checkpoint is not None else op_checkpoint8(input, seed)) if compress else x
        saved = LinearSaved(kept, zc if zc is not None else z, weight, activation, shape, out_shape, dtype, bias is not None)
    if rows == 0:
        return y, saved
    guard, stream = nv.guard_and_stream(x)
    with guard:
        xk, xp, xld = _operand(x, rows, cin, ld, stream)
        w, _, wld = _rows(weight, cin)
        wk, wp, wld = _operand(w, cout, cin, wld, stream)
        nbytes = _LIB.gact_linear_scratch_bytes(rows, cin, cout, 0)
        scratch = _scratch(nbytes, dev)
        # codes of the pre-activation draw their noise from the next seed
        nv.check(_LIB.gact_linear(xp, xld, wp, wld, _ptr(bias), _ptr(res), ld_res, nv.DTYPE_CODE[dtype], rows, cin, cout, act, y.data_ptr(),
                                  _ptr(z), None if zc is None else zc.codes.data_ptr(), None if zc is None else zc.scales.data_ptr(), stoch,
                                  (s + 0x9E3779B97F4A7C15) & 0xFFFFFFFFFFFFFFFF, _ptr(scratch), stream), "gact_linear")
    _count(1 + (nbytes > 0))
    return y, saved


def op_linear_backward(grad_output, saved, needs=(True, True, True)):
    """(grad of the input, of weight, of bias) from what op_linear saved; None where ``needs`` says so or there is no bias.
    The gradient of a residual is grad_output itself."""
    cout, cin = saved.weight.shape
    dtype = saved.dtype
    _check_tensor(grad_output, "grad_output", (dtype,), like=saved.weight)
    if grad_output.shape != saved.out_shape:
        raise ValueError("grad_output must have shape %s, got %s" % (tuple(saved.out_shape), tuple(grad_output.shape)))
    need_x, need_w, need_b = needs[0], needs[1], needs[2] and saved.has_bias
    dy, rows, ld = _rows(grad_output, cout)
    dev = dy.device
    act, code = nv.ACT_CODE[saved.activation], nv.DTYPE_CODE[dtype]
    dx = torch.empty(saved.in_shape, dtype=dtype, device=dev) if need_x else None
    dw = torch.empty((cout, cin), dtype=dtype, device=dev) if need_w else None
    db = torch.empty(cout, dtype=dtype, device=dev) if need_b else None
    if rows == 0:
        return dx, (None if dw is None else dw.zero_()), (None if db is None else db.zero_())
    guard, stream = nv.guard_and_stream(dy)
    with guard:
        dz, ld_dz = dy, ld
        if act or need_b:
            z, zld, zc = None, 0, None
            if act:
                if isinstance(saved.z, Checkpoint8):
                    zc = saved.z
                    _check_checkpoint(zc, cout, rows, dy, "saved pre-activation")
                else:
                    z, _, zld = _rows(saved.z, cout)
                ld_dz = (cout + 7) // 8 * 8
                dz = torch.empty((rows, ld_dz), dtype=dtype, device=dev)
            scratch = _scratch(_LIB.gact_act_backward_scratch_bytes(rows, cout), dev) if need_b else None
            nv.check(_LIB.gact_act_backward(dy.data_ptr(), code, rows, cout, ld, act, _ptr(z), zld,
                                            None if zc is None else zc.codes.data_ptr(), None if zc is None else zc.scales.data_ptr(),
                                            dz.data_ptr() if act else None, ld_dz, _ptr(db), _ptr(scratch), stream), "gact_act_backward")
            _count(1 + need_b)
        if need_x or need_w:
            dzk, dzp, ld_dz = _operand(dz, rows, cout, ld_dz, stream)
        if need_x:
            w, _, wld = _rows(saved.weight, cin)
            wk, wp, wld = _operand(w, cout, cin, wld, stream)
            nbytes = _LIB.gact_linear_scratch_bytes(rows, cin, cout, 1)
            scratch = _scratch(nbytes, dev)
            nv.check(_LIB.gact_linear_dgrad(dzp, ld_dz, wp, wld, code, rows, cin, cout, dx.data_ptr(), _ptr(scratch), stream), "gact_linear_dgrad")
            _count(1 + (nbytes > 0))
        if need_w:
            if isinstance(saved.x, Checkpoint8):
                c = saved.x
                _check_checkpoint(c, cin, rows, dy, "saved input")
                xld = c.codes.shape[1]
                xk = torch.empty((rows, xld), dtype=dtype, device=dev)
                nv.check(_LIB.gact_restore8(c.codes.data_ptr(), c.scales.data_ptr(), rows, cin, code, xk.data_ptr(), xld, stream), "gact_restore8")
                _count(1)
                xp = xk.data_ptr()
            else:
                x, _, xld = _rows(saved.x, cin)
                xk, xp, xld = _operand(x, rows, cin, xld, stream)
            nbytes = _LIB.gact_linear_scratch_bytes(rows, cin, cout, 2)
            scratch = _scratch(nbytes, dev)
            nv.check(_LIB.gact_linear_wgrad(dzp, ld_dz, xp, xld, code, rows, cin, cout, dw.data_ptr(), _ptr(scratch), stream), "gact_linear_wgrad")
            _count(1 + (nbytes > 0))
    return dx, dw, db
