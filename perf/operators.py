"""The training operators with 8-bit activation checkpoints: what is measured, and their plain forms.

Three operators, each case one pass as a training step makes it:

``checkpoint``  x is kept as 8-bit codes with a power-of-two scale for every 32 elements of a row, and restored;
``layer_norm``  forward, then backward from the 8-bit codes of x (or from x itself), weight and bias gradients reduced;
``linear``      y = act(x W^T + b) + residual forward, then the gradients of x, W and b from the 8-bit codes of x and of
                the pre-activation (or from the tensors themselves).

With ``own`` false the passes run in elementary torch operations in 32 bits, with ``own`` true through ``gact.fused``.
"""
import math
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parents[1]
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ITEM = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = 32


def _fused():
    path = str(ROOT / "gact-icml_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from gact import fused
    return fused


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def _ck(name, rows, cols, dtype):
    return {"name": name, "op": "checkpoint", "rows": rows, "cols": cols, "dtype": dtype}


def _ln(name, rows, cols, dtype, compress=True):
    return {"name": name, "op": "layer_norm", "rows": rows, "cols": cols, "dtype": dtype, "compress": compress}


def _lin(name, rows, cin, cout, dtype, act="none", residual=False, compress=True):
    return {"name": name, "op": "linear", "rows": rows, "cin": cin, "cout": cout, "dtype": dtype, "act": act,
            "residual": residual, "compress": compress}


def listed():
    return [
        # the hidden states of the 8 samples (seq 128) that the sensitivity probe of BERT-large runs on
        _ck("checkpoint_probe_hidden", 1024, 1024, "bf16"),
        # ragged rows of an fp32 model
        _ck("checkpoint_odd_f32", 8191, 1003, "f32"),
        # the feed-forward activations of a BERT-large batch of 512 sequences of 128 tokens
        _ck("checkpoint_large", 65536, 4096, "bf16"),
        # one sequence of 128 tokens: latency counts
        _ln("norm_one_sequence", 128, 1024, "bf16"),
        # BERT-large's layer norm at its training batch (64 x 128 tokens)
        _ln("norm_bert_large", 8192, 1024, "bf16"),
        # fp32 rows of odd length, as layer norm runs under autocast
        _ln("norm_odd_f32", 10007, 771, "f32"),
        # long rows, many tokens
        _ln("norm_large", 65536, 4096, "bf16"),
        # the classification head of BERT-large: two labels
        _lin("linear_classifier", 64, 1024, 2, "bf16"),
        # ragged everything, fp16
        _lin("linear_odd_f16", 1000, 771, 333, "f16", "gelu", True),
        # BERT-large's feed-forward pair at its training batch
        _lin("linear_ffn_up", 8192, 1024, 4096, "bf16", "gelu"),
        _lin("linear_ffn_down", 8192, 4096, 1024, "bf16", "none", True),
        # the same width at a batch of 256 sequences
        _lin("linear_large", 32768, 4096, 4096, "bf16", "gelu", True),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of lo .. hi."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """Like _log; half of the draws are rounded to a multiple of 8 where that is possible, the others stay as they fall."""
    n = _log(rng, lo, hi)
    return max(lo, n // 8 * 8) if rng.random() < 0.5 and n >= 8 else n


def draw(rng):
    op = rng.choice(["checkpoint", "layer_norm", "linear"])
    if op == "linear":
        c = _lin("", _size(rng, 1, 32768), _size(rng, 1, 4096), _size(rng, 1, 4096), rng.choice(["bf16", "f16"]),
                 rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), rng.random() < 0.5, rng.random() < 0.8)
    else:
        # a norm over a handful of elements is all cancellation: its rows start at 16
        rows, cols = _size(rng, 1, 65536), _size(rng, 1 if op == "checkpoint" else 16, 8192)
        dtype = rng.choice(["bf16", "f16", "f32"])
        rows = min(rows, 65536 * 4096 // cols // (2 if dtype == "f32" else 1))      # no more than the largest listed one
        c = _ck("", rows, cols, dtype) if op == "checkpoint" else _ln("", rows, cols, dtype, rng.random() < 0.8)
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dt):
        out = torch.empty(shape, dtype=dtype, device="cuda")
        return out.normal_(0.0, std, generator=g)

    if case["op"] == "linear":
        m, k, n = case["rows"], case["cin"], case["cout"]
        s = {"case": dict(case), "x": normal(m, k), "w": normal(n, k, std=1.0 / math.sqrt(k)), "b": normal(n, std=0.1),
             "dy": normal(m, n, std=0.05)}
        s["res"] = normal(m, n) if case["residual"] else None
        return s
    m, h = case["rows"], case["cols"]
    # activations: unequal scales from channel to channel, a few of them large
    chan = torch.empty(h, device="cuda").normal_(0.0, 1.0, generator=g).mul_(0.5).exp_()
    x = normal(m, h).mul_(chan.to(dt))
    s = {"case": dict(case), "x": x}
    if case["op"] == "layer_norm":
        x.add_(normal(h, std=0.1))
        s["w"] = normal(h, std=0.1).add_(1.0)
        s["b"] = normal(h, std=0.1)
        s["dy"] = normal(m, h, std=0.05)
        s["eps"] = 1e-5
    return s


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    fused, c = _fused(), s["case"]
    if c["op"] == "checkpoint":
        return fused.op_restore8(fused.op_checkpoint8(s["x"]))
    if c["op"] == "layer_norm":
        y, saved = fused.op_layer_norm(s["x"], s["w"], s["b"], s["eps"], compress=c["compress"])
        dx, dw, db = fused.op_layer_norm_backward(s["dy"], saved)
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    act = None if c["act"] == "none" else c["act"]
    y, saved = fused.op_linear(s["x"], s["w"], s["b"], activation=act, residual=s["res"], compress=c["compress"])
    dx, dw, db = fused.op_linear_backward(s["dy"], saved)
    return {"y": y, "dx": dx, "dw": dw, "db": db}


def _plain_kept(x, positive=False):
    """The values that the 8-bit checkpoint of x (fp32, rows x cols) stands for.  ``positive``: a value above zero keeps a
    code above zero (the checkpoint of a ReLU's pre-activation)."""
    m, k = x.shape
    kp = (k + BLOCK - 1) // BLOCK * BLOCK
    v = torch.nn.functional.pad(x, (0, kp - k)).view(m, kp // BLOCK, BLOCK)
    top = v.abs().amax(dim=2, keepdim=True)
    # biased exponent of the scale: the largest magnitude of the block falls into [63.5, 127) steps
    e = torch.clamp(((top.view(torch.int32) + 0x20000) >> 23) - 6, min=1)
    scale = torch.where(torch.isfinite(top), (e.clamp(max=254) << 23).view(torch.float32), torch.full_like(top, math.nan))
    up = ((254 - e.clamp(max=253)) << 23).view(torch.float32)
    code = torch.round(v * up)
    if positive:
        code = torch.where(v > 0, code.clamp(min=1.0), code)
    return (code * scale).view(m, kp)[:, :k]


def _plain_act(z, act):
    if act == "none":
        return z
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    return z / (1.0 + torch.exp(-z))


def _plain_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z)
    s = 1.0 / (1.0 + torch.exp(-z))
    return s * (1.0 + z * (1.0 - s))


def _run_plain(s):
    c, x = s["case"], s["x"]
    dt, xf = x.dtype, x.float()
    if c["op"] == "checkpoint":
        return _plain_kept(xf).to(dt)
    if c["op"] == "layer_norm":
        w, b, dy = s["w"].float(), s["b"].float(), s["dy"].float()
        mean = xf.mean(dim=1, keepdim=True)
        cent = xf - mean
        r = 1.0 / torch.sqrt((cent * cent).mean(dim=1, keepdim=True) + s["eps"])
        y = cent * r * w + b
        xh = ((_plain_kept(xf) if c["compress"] else xf) - mean) * r
        g = dy * w
        dx = r * (g - g.mean(dim=1, keepdim=True) - xh * (g * xh).mean(dim=1, keepdim=True))
        return {"y": y.to(dt), "dx": dx.to(dt), "dw": (dy * xh).sum(dim=0).to(dt), "db": dy.sum(dim=0).to(dt)}
    act, w, dy = c["act"], s["w"].float(), s["dy"].float()
    z = xf @ w.t() + s["b"].float()
    y = _plain_act(z, act)
    if s["res"] is not None:
        y = y + s["res"].float()
    y = y.to(dt)
    if act == "none":
        dz = dy
    else:
        # without compression the pre-activation is kept in the type of the inputs
        dz = dy * _plain_slope(_plain_kept(z, act == "relu") if c["compress"] else z.to(dt).float(), act)
    dx = dz @ w
    dw = dz.t() @ (_plain_kept(xf) if c["compress"] else xf)
    return {"y": y, "dx": dx.to(dt), "dw": dw.to(dt), "db": dz.sum(dim=0).to(dt)}


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def _kept_bytes(rows, cols):
    blocks = (cols + BLOCK - 1) // BLOCK
    return rows * blocks * (BLOCK + 1)


def work(case):
    it = ITEM[case["dtype"]]
    if case["op"] == "checkpoint":
        # read x, write codes and scales; read them, write the restored tensor
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * n * it + 2 * _kept_bytes(case["rows"], case["cols"]), "flops": 4 * n}
    if case["op"] == "layer_norm":
        n, h = case["rows"] * case["cols"], case["cols"]
        # forward: x in, y out; backward: dy in, dx out; what is kept between the two is written and read once
        # (x itself is already there where nothing is compressed: it is read again); w twice, b, dw, db
        kept = 2 * _kept_bytes(case["rows"], h) if case["compress"] else n * it
        return {"bytes": 4 * n * it + kept + 16 * case["rows"] + 5 * h * it, "flops": 20 * n}
    m, k, n = case["rows"], case["cin"], case["cout"]
    # x, W, b, dy in, y, dx, dW, db out (W is read by both directions), the residual, and what is kept
    b = it * (2 * m * k + 3 * n * k + 2 * m * n + 2 * n + (m * n if case["residual"] else 0))
    if case["compress"]:
        b += 2 * _kept_bytes(m, k) + (2 * _kept_bytes(m, n) if case["act"] != "none" else 0)
    else:
        b += it * (m * k + (2 * m * n if case["act"] != "none" else 0))
    return {"bytes": b, "flops": 6 * m * n * k}


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def _exact_kept(x, positive=False):
    """Blocks of 32, step 2^s with the smallest s >= -126 for which max|x| < 127 * 2^s (so a step is a power of two and
    every code fits 7 bits and a sign); nearest code, ties to even; a block that holds NaN or infinity is NaN."""
    rows, cols = x.shape
    out = torch.empty_like(x)
    whole = cols // BLOCK * BLOCK
    parts = [(0, whole, BLOCK)] if whole else []
    if cols > whole:
        parts.append((whole, cols, cols - whole))
    for lo, hi, width in parts:
        v = x[:, lo:hi].reshape(rows, -1, width)
        top = v.abs().amax(dim=2, keepdim=True)
        frac, ex = torch.frexp(top / 127.0)                     # top = 127 * frac * 2^ex, frac in [0.5, 1)
        # the smallest power of two ABOVE top / 127 (at a power of two itself the next one)
        s = torch.where(top > 0, ex, torch.full_like(ex, -126)).clamp(min=-126)
        step = torch.ldexp(torch.ones_like(top), s)
        q = torch.round(v / step)
        if positive:
            q = torch.where((v > 0) & (q < 1), torch.ones_like(q), q)
        q = torch.where(torch.isfinite(top), q * step, torch.full_like(v, math.nan))
        out[:, lo:hi] = q.reshape(rows, hi - lo)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"] == "checkpoint":
        return _exact_kept(x)
    if case["op"] == "layer_norm":
        w, b, dy = s["w"].double(), s["b"].double(), s["dy"].double()
        var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        std = (var + s["eps"]).sqrt()
        y = torch.addcmul(b, (x - mean) / std, w)
        xh = (x if not case["compress"] else _exact_kept(x)).sub(mean).div(std)
        h = case["cols"]
        g = dy * w
        # the Jacobian of the normalisation applied to g
        dx = (g - (g.sum(1, keepdim=True) + xh * (g * xh).sum(1, keepdim=True)) / h) / std
        return {"y": y, "dx": dx, "dw": torch.einsum("ij,ij->j", dy, xh), "db": torch.einsum("ij->j", dy)}
    act = case["act"]
    w, dy = s["w"].double(), s["dy"].double()
    z = torch.addmm(s["b"].double(), x, w.t())
    kept = _exact_kept(z, act == "relu") if case["compress"] else z.to(s["x"].dtype).double()

    def f(t):
        """(value, derivative) of the activation."""
        if act == "relu":
            return t.clamp(min=0.0), (t > 0).double()
        if act == "gelu":
            cdf = 0.5 * torch.erfc(-t / math.sqrt(2.0))
            return t * cdf, cdf + t * torch.exp(-t * t / 2) / math.sqrt(2.0 * math.pi)
        if act == "gelu_tanh":
            a = math.sqrt(2.0 / math.pi)
            # (1 + tanh u) / 2 = sigmoid(2u)
            p = torch.sigmoid(2 * a * (t + 0.044715 * t ** 3))
            return t * p, p + t * p * (1 - p) * 2 * a * (1 + 0.134145 * t * t)
        if act == "silu":
            p = torch.sigmoid(t)
            return t * p, p + t * p * (1 - p)
        return t, torch.ones_like(t)

    y = f(z)[0]
    if s["res"] is not None:
        y = y + s["res"].double()
    del z
    dz = dy * f(kept)[1]
    del kept
    dw = torch.mm(dz.t(), _exact_kept(x) if case["compress"] else x)
    return {"y": y, "dx": torch.mm(dz, w), "dw": dw, "db": torch.einsum("ij->j", dz)}
