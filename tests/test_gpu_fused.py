"""The training operators with 8-bit activation checkpoints (gact.fused) against their formulas in 64 bits.

Tolerances are bounds, worked out before the first run: a stored value is off by half a step of its type
(finfo.eps / 2, relative); an fp32 sum of n terms by n * 2^-24 of the sum of magnitudes (2^-23 for the tensor cores, whose
adder may truncate); checkpoints are exact.
"""
import math

import pytest
import torch

gpu = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U24, U23 = 2.0 ** -24, 2.0 ** -23


def half_step(t):
    return torch.finfo(t).eps / 2


def kept64(x, positive=False):
    """The values a checkpoint of x stands for, from the definition, in 64 bits on the CPU."""
    x = x.detach().double().cpu()
    cols = x.shape[-1]
    flat = x.reshape(-1, cols)
    out = torch.empty_like(flat)
    for lo in range(0, cols, 32):
        v = flat[:, lo:lo + 32]
        top = v.abs().amax(dim=1, keepdim=True)
        s = torch.frexp(top / 127.0)[1].clamp(min=-126)
        s = torch.where(top > 0, s, torch.full_like(s, -126))
        step = torch.ldexp(torch.ones_like(top), s)
        q = torch.round(v / step)
        if positive:
            q = torch.where((v > 0) & (q < 1), torch.ones_like(q), q)
        out[:, lo:lo + 32] = torch.where(torch.isfinite(top), q * step, torch.full_like(v, math.nan))
    return out.reshape(x.shape)


def inputs(*shape, dtype, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(dtype)


def within(got, want, tol, what):
    got, want = got.detach().double().cpu(), want.double().cpu()
    assert got.shape == want.shape, what
    bad = (got - want).abs() > tol.double().cpu()
    assert not bad.any() and not got.isnan().any(), "%s: %d of %d off, worst by %g over its bound" % (
        what, int(bad.sum()), bad.numel(), float(((got - want).abs() - tol.double().cpu()).max()))


def same(got, want):
    return torch.equal(torch.nan_to_num(got.double().cpu(), nan=12345.0), torch.nan_to_num(want.double().cpu(), nan=12345.0))


# ---------------------------------------------------------------------------------------------------------------
# checkpoints
# ---------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(1, 1), (1, 31), (3, 32), (7, 33), (5, 1, 64), (1000, 8), (77, 1003), (300, 4096), (2, 3, 5, 100), (40000, 40), (17,),
                                   (3, 8, 70000)])
def test_checkpoint_is_exact(shape, dtype):
    from gact import fused
    x = inputs(*shape, dtype=DT[dtype], seed=sum(shape))
    x.view(-1)[::7] *= 30.0
    c = fused.op_checkpoint8(x)
    cols = shape[-1]
    pitch = (cols + 31) // 32 * 32
    rows = x.numel() // cols
    assert c.codes.shape == (rows, pitch) and c.scales.shape == (rows, pitch // 32)
    assert int(c.codes[:, cols:].abs().sum()) == 0 and int(c.codes.min()) >= -127
    y = fused.op_restore8(c)
    assert y.shape == x.shape and y.dtype == x.dtype
    assert same(y, kept64(x))
    assert same(fused.op_restore8(c, torch.float32), kept64(x))


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_checkpoint_of_special_values(dtype):
    from gact import fused
    dt = DT[dtype]
    top = torch.finfo(dt).max
    rows = [
        [0.0] * 40,
        [-0.0] * 40,
        [127.0] + [1.0] * 39,                      # exactly 127 steps of 1: the scale doubles
        [126.5] + [0.5] * 39,
        [63.5, -63.5] + [0.25] * 38,
        [float("nan")] + [1.0] * 39,               # first block only
        [1.0] * 35 + [float("inf")] + [2.0] * 4,   # short block only
        [torch.finfo(dt).tiny] * 40,
        [torch.finfo(dt).tiny / 4] * 40,           # subnormal
        [1e-3 * (-1) ** i for i in range(40)],
    ]
    x = torch.tensor(rows, dtype=torch.float64).to(dt).cuda()
    y = fused.op_restore8(fused.op_checkpoint8(x))
    assert same(y, kept64(x))
    assert y[5, :32].isnan().all() and not y[5, 32:].isnan().any()
    assert y[6, 32:].isnan().all() and not y[6, :32].isnan().any()
    # the highest binade stays finite: 63 of its steps instead of 64
    z = torch.tensor([[top, -top, 1.0, 0.0] * 8], dtype=dt, device="cuda")
    w = fused.op_restore8(fused.op_checkpoint8(z))
    assert w.isfinite().all() and bool(((w - z).double().abs() <= top / 64 * 1.01).all())


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_checkpoint_of_strided_and_misaligned_rows(dtype):
    from gact import fused
    big = inputs(50, 1000, dtype=DT[dtype], seed=3)
    for x in (big[:, 3:700], big[::2, :512], big[:, :1], big.t(), big[:, 8:264], big.reshape(-1)[1:50 * 999 + 1].view(50, 999),
              big[:1].expand(9, 1000), big.view(5, 10, 1000).transpose(0, 1), big.view(5, 10, 1000)[:, 2:7, 16:48]):
        c = fused.op_checkpoint8(x)
        assert same(fused.op_restore8(c), kept64(x))


@gpu
def test_checkpoint_of_nothing():
    from gact import fused
    for shape in ((0, 64), (4, 0), (0,), (2, 0, 32)):
        y = fused.op_restore8(fused.op_checkpoint8(torch.empty(shape, device="cuda", dtype=torch.bfloat16)))
        assert y.shape == torch.Size(shape)


def philox7(counter, seed):
    """Philox4x32 with 7 rounds on Python integers."""
    c = [counter & 0xffffffff, counter >> 32, 0, 0]
    k0, k1 = seed & 0xffffffff, seed >> 32
    for _ in range(7):
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(p1 >> 32) ^ c[1] ^ k0, p1 & 0xffffffff, (p0 >> 32) ^ c[3] ^ k1, p0 & 0xffffffff]
        k0, k1 = (k0 + 0x9E3779B9) & 0xffffffff, (k1 + 0xBB67AE85) & 0xffffffff
    return c


@gpu
def test_stochastic_codes_match_the_generator_and_are_unbiased():
    from gact import fused
    x = inputs(6, 71, dtype=torch.float32, seed=11)
    seed = 0x123456789ABCDEF
    c = fused.op_checkpoint8(x, seed=seed)
    assert torch.equal(c.codes, fused.op_checkpoint8(x, seed=seed).codes)
    assert not torch.equal(c.codes, fused.op_checkpoint8(x, seed=seed + 1).codes)
    codes, scales, xs = c.codes.cpu(), c.scales.cpu().view(torch.uint8), x.cpu().double()
    for r in range(6):
        for col in range(71):
            i = r * 96 + col
            w = philox7(i // 8, seed)[(i % 8) // 2]
            u = (((w >> 16) if i & 1 else (w & 0xffff)) + 0.5) / 65536
            v = float(xs[r, col]) * 2.0 ** (127 - int(scales[r, col // 32]))
            assert int(codes[r, col]) in (math.floor(v + u), math.floor(float(torch.tensor(v + u, dtype=torch.float32)))), (r, col)
    # the mean over many seeds approaches x: standard error of a code is at most 0.5 / sqrt(n)
    n = 4000
    y = torch.zeros_like(x, dtype=torch.float64)
    for s in range(n):
        y += fused.op_restore8(fused.op_checkpoint8(x, seed=s)).double()
    step = torch.ldexp(torch.ones(6, 3, dtype=torch.float64), scales.int() - 127).repeat_interleave(32, 1)[:, :71]
    assert bool(((y.cpu() / n - xs).abs() / step).max() < 6 * 0.5 / math.sqrt(n))


# ---------------------------------------------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------------------------------------------
def check_norm(x, w, b, dy, eps, compress, needs=(True, True, True)):
    from gact import fused
    y, saved = fused.op_layer_norm(x, w, b, eps, compress=compress)
    got = fused.op_layer_norm_backward(dy, saved, needs)
    cols = x.shape[-1]
    x64 = x.double().cpu().reshape(-1, cols)
    w64 = torch.ones(cols, dtype=torch.float64) if w is None else w.double().cpu()
    b64 = torch.zeros(cols, dtype=torch.float64) if b is None else b.double().cpu()
    dy64 = dy.double().cpu().reshape(-1, cols)
    mean = x64.mean(1, keepdim=True)
    r = 1.0 / torch.sqrt(x64.var(1, unbiased=False, keepdim=True) + eps)
    xh = (x64 - mean) * r
    # an fp32 error of a few steps of x and of the mean (a sum of up to 64 terms one after the other), seen through r
    err = 64 * U24 * ((x64.abs() + x64.abs().mean(1, keepdim=True)) * r + xh.abs())
    ref = xh * w64 + b64
    h = half_step(x.dtype)
    tiny = torch.finfo(x.dtype).tiny
    within(y.reshape(-1, cols), ref, h * 1.01 * ref.abs() + 1.01 * err * w64.abs() + 4 * U24 * b64.abs() + tiny, "y")
    xk = kept64(x).reshape(-1, cols) if compress else x64
    xk_h = (xk - mean) * r
    err = 64 * U24 * ((xk.abs() + x64.abs() + 2 * x64.abs().mean(1, keepdim=True)) * r + xk_h.abs())
    g = dy64 * w64
    c1, c2 = g.mean(1, keepdim=True), (g * xk_h).mean(1, keepdim=True)
    dx = r * (g - c1 - xk_h * c2)
    e1 = 64 * U24 * g.abs().mean(1, keepdim=True)
    e2 = 64 * U24 * (g * xk_h).abs().mean(1, keepdim=True) + (g.abs() * err).mean(1, keepdim=True)
    tol = h * 1.01 * dx.abs() + r * (8 * U24 * (g.abs() + c1.abs() + (xk_h * c2).abs()) + e1 + xk_h.abs() * e2 + err * (c2.abs() + e2)) + 1e-30
    rows = x64.shape[0]
    k = (64 + rows / 64) * U24
    pt = w.dtype if w is not None else b.dtype if b is not None else x.dtype
    hp = half_step(pt)
    dw = (dy64 * xk_h).sum(0)
    db = dy64.sum(0)
    if needs[0]:
        within(got[0].reshape(-1, cols), dx, tol + tiny, "dx")
    if needs[1]:
        within(got[1], dw, hp * 1.01 * dw.abs() + k * (dy64 * xk_h).abs().sum(0) + 1.01 * (dy64.abs() * err).sum(0) + 1e-30 + torch.finfo(pt).tiny, "dw")
    if needs[2]:
        within(got[2], db, hp * 1.01 * db.abs() + k * dy64.abs().sum(0) + 1e-30 + torch.finfo(pt).tiny, "db")
    assert [t is not None for t in got] == list(needs)
    return y, got


NORM_SHAPES = [(1, 1), (1, 7), (3, 32), (5, 33), (300, 64), (65, 100), (129, 128), (33, 256), (40, 257), (70, 512), (9, 771), (130, 1024), (2000, 1024), (21, 1500),
               (20, 2048), (11, 2049), (31, 4096), (7, 8192), (6, 5001), (3, 8200), (3, 16384), (2, 3, 4, 96), (4099, 16)]


@gpu
@pytest.mark.parametrize("compress", [True, False])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", NORM_SHAPES)
def test_layer_norm(shape, dtype, compress):
    dt = DT[dtype]
    cols = shape[-1]
    x = inputs(*shape, dtype=dt, seed=1) * 2 + 0.5
    w, b = inputs(cols, dtype=dt, seed=2, std=0.2) + 1, inputs(cols, dtype=dt, seed=3, std=0.3)
    check_norm(x, w, b, inputs(*shape, dtype=dt, seed=4, std=0.1), 1e-5, compress)


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_layer_norm_parameters(dtype):
    """fp32 weights with 16-bit rows, missing weight or bias, every subset of gradients."""
    dt = DT[dtype]
    x, dy = inputs(100, 200, dtype=dt, seed=1), inputs(100, 200, dtype=dt, seed=4, std=0.1)
    w, b = inputs(200, dtype=torch.float32, seed=2) + 1, inputs(200, dtype=torch.float32, seed=3)
    for compress in (True, False):
        check_norm(x, w, b, dy, 1e-12, compress)
        check_norm(x, w, None, dy, 1e-5, compress)
        check_norm(x, None, b, dy, 1e-5, compress)
        check_norm(x, None, None, dy, 1e-5, compress)
        for needs in ((True, False, False), (False, True, False), (False, False, True), (False, True, True), (True, False, True), (True, True, False)):
            check_norm(x, w, b, dy, 1e-5, compress, needs)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_layer_norm_strides(dtype):
    dt = DT[dtype]
    big, gy = inputs(60, 900, dtype=dt, seed=5), inputs(60, 900, dtype=dt, seed=6, std=0.1)
    w, b = inputs(900, dtype=dt, seed=7) + 1, inputs(900, dtype=dt, seed=8)
    for cut in (lambda t: t[:, 1:400], lambda t: t[::3, 8:264], lambda t: t.t()[:100], lambda t: t[:1].expand(7, 900),
                lambda t: t.view(6, 10, 900).transpose(0, 1)):
        x, dy = cut(big), cut(gy)
        n = x.shape[-1]
        check_norm(x, w[:n], b[1:n + 1] if n < 900 else b, dy, 1e-5, True)
        check_norm(x, w[:n], b[:n], dy, 1e-5, False)


@gpu
def test_layer_norm_special_rows():
    """Constant rows (variance 0) give the bias; a NaN or an infinity stays in its row of y; no rows give zero gradients."""
    from gact import fused
    x = inputs(6, 96, dtype=torch.bfloat16, seed=1)
    x[1] = 3.0
    x[2, 5], x[3, 70] = float("nan"), float("inf")
    w, b = inputs(96, dtype=torch.bfloat16, seed=2), inputs(96, dtype=torch.bfloat16, seed=3)
    y, saved = fused.op_layer_norm(x, w, b)
    assert torch.equal(y[1], b) and y[2].isnan().all() and y[3].isnan().all()
    assert y[[0, 1, 4, 5]].isfinite().all()
    dx, dw, db = fused.op_layer_norm_backward(torch.ones_like(x), saved)
    assert dx[[0, 1, 4, 5]].isfinite().all() and dx[2].isnan().any() and db.isfinite().all() and bool((db == 6).all())
    for compress in (True, False):
        y, saved = fused.op_layer_norm(x[:0], w, b, compress=compress)
        dx, dw, db = fused.op_layer_norm_backward(y, saved)
        assert y.shape == dx.shape == (0, 96) and bool((dw == 0).all()) and bool((db == 0).all())
    y, saved = fused.op_layer_norm(x, w, b, save=False)
    assert saved is None


# ---------------------------------------------------------------------------------------------------------------
# linear
# ---------------------------------------------------------------------------------------------------------------
def act64(t, act):
    """(value, slope) in 64 bits."""
    if act == "relu":
        return t.clamp(min=0), (t > 0).double()
    if act == "gelu":
        c = 0.5 * torch.erfc(-t / math.sqrt(2))
        return t * c, c + t * torch.exp(-t * t / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        a = math.sqrt(2 / math.pi)
        th = torch.tanh(a * (t + 0.044715 * t ** 3))
        return 0.5 * t * (1 + th), 0.5 * (1 + th) + 0.5 * t * (1 - th ** 2) * a * (1 + 3 * 0.044715 * t * t)
    if act == "silu":
        p = torch.sigmoid(t)
        return t * p, p * (1 + t * (1 - p))
    return t, torch.ones_like(t)


def check_linear(x, w, b, act, res, dy, compress, needs=(True, True, True), checkpoint=None):
    from gact import fused
    y, saved = fused.op_linear(x, w, b, activation=act, residual=res, compress=compress, checkpoint=checkpoint)
    got = fused.op_linear_backward(dy, saved, needs)
    cout, cin = w.shape
    d = lambda t: t.double().cpu()
    x64, w64, dy64 = d(x).reshape(-1, cin), d(w), d(dy).reshape(-1, cout)
    b64 = torch.zeros(cout, dtype=torch.float64) if b is None else d(b)
    rows = x64.shape[0]
    h = half_step(x.dtype)
    tiny = torch.finfo(x.dtype).tiny
    z = x64 @ w64.t() + b64
    err_z = (cin + 8) * U23 * (x64.abs() @ w64.abs().t() + b64.abs())
    ref = act64(z, act)[0]
    if res is not None:
        ref = ref + d(res).reshape(-1, cout)
    # slopes are below 1.13; the approximations of Phi and the exponentials are good to 1e-6 of the value's scale
    within(y.reshape(-1, cout), ref, h * 1.01 * ref.abs() + 1.2 * err_z + 2e-6 * z.abs() + 4 * U24 * ref.abs() + tiny, "y")
    # the pre-activation as it was kept
    if act is not None:
        if compress:
            zk = d(fused.op_restore8(saved.z, torch.float32)).reshape(-1, cout)
            n32 = (cout + 31) // 32 * 32
            top = torch.nn.functional.pad(z.abs() + err_z, (0, n32 - cout)).reshape(rows, -1, 32).amax(2).repeat_interleave(32, 1)[:, :cout]
            # half a step of the block (a whole one for a positive value that ReLU keeps above zero)
            within(zk, z, top / 63.5 * (1.0 if act == "relu" else 0.5) + err_z + 1e-37, "kept z")
            if act == "relu":
                sure = z.abs() > err_z
                assert bool(((zk > 0) == (z > 0))[sure].all())
        else:
            zk = d(saved.z)
            within(zk, z, h * 1.01 * z.abs() + 1.01 * err_z + tiny, "kept z")
        slope = act64(zk, act)[1]
    else:
        slope = torch.ones_like(dy64)
    dz = dy64 * slope
    err_s = 4e-6 * dy64.abs() if act not in (None, "relu") else torch.zeros_like(dz)
    err_dz = err_s + (h * 1.01 * dz.abs() + tiny if act is not None else 0)
    if needs[0]:
        dx = dz @ w64
        mag = dz.abs() @ w64.abs()
        within(got[0].reshape(-1, cin), dx, h * 1.01 * dx.abs() + (cout + 8) * U23 * mag + 1.01 * err_dz @ w64.abs() + tiny if act is not None
               else h * 1.01 * dx.abs() + (cout + 8) * U23 * mag + tiny, "dx")
    if needs[1]:
        xk = kept64(x).reshape(-1, cin) if compress else x64
        dw = dz.t() @ xk
        mag = dz.abs().t() @ xk.abs()
        tol = h * 1.01 * dw.abs() + (rows + 8) * U23 * mag + tiny
        if act is not None:
            tol = tol + 1.01 * err_dz.t() @ xk.abs()
        within(got[1], dw, tol, "dw")
    if needs[2] and b is not None:
        db = dz.sum(0)
        within(got[2], db, h * 1.01 * db.abs() + (64 + rows / 64) * U24 * dz.abs().sum(0) + err_s.sum(0) + tiny, "db")
    assert [t is not None for t in got] == [needs[0], needs[1], needs[2] and b is not None]
    return y, got


LINEAR_SIZES = [(1, 1, 1), (1, 8, 8), (5, 3, 7), (2, 64, 256), (128, 64, 256), (129, 65, 257), (300, 1024, 2), (64, 40, 1000), (1000, 771, 333), (640, 512, 768),
                (1, 1024, 1024), (17, 4096, 64), (4000, 96, 33), (513, 1024, 1024), (130, 192, 4096)]


@gpu
@pytest.mark.parametrize("compress", [True, False])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("size", LINEAR_SIZES)
def test_linear(size, dtype, compress):
    m, k, n = size
    dt = DT[dtype]
    x, w = inputs(m, k, dtype=dt, seed=1), inputs(n, k, dtype=dt, seed=2, std=1 / math.sqrt(k))
    b, res, dy = inputs(n, dtype=dt, seed=3, std=0.3), inputs(m, n, dtype=dt, seed=4), inputs(m, n, dtype=dt, seed=5, std=0.1)
    check_linear(x, w, b, None, None, dy, compress)
    check_linear(x, w, b, "gelu", res, dy, compress)


@gpu
@pytest.mark.parametrize("act", [None, "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("compress", [True, False])
def test_linear_epilogues(act, compress):
    m, k, n = 200, 136, 264
    dt = torch.bfloat16
    x, w = inputs(m, k, dtype=dt, seed=1), inputs(n, k, dtype=dt, seed=2, std=0.3)
    b, res, dy = inputs(n, dtype=dt, seed=3), inputs(m, n, dtype=dt, seed=4), inputs(m, n, dtype=dt, seed=5, std=0.1)
    for bias in (b, None):
        for r in (res, None):
            check_linear(x, w, bias, act, r, dy, compress)
    for needs in ((True, False, False), (False, True, False), (False, False, True), (False, False, False)):
        check_linear(x, w, b, act, None, dy, compress, needs)


@gpu
@pytest.mark.parametrize("size", [(5, 3, 7), (70, 40, 33), (300, 1024, 2)])
def test_linear_without_bias_and_with_odd_outputs(size):
    """No activation and no bias: the gradient itself is the products' operand, copied to 16-byte rows where it has none."""
    m, k, n = size
    x, w, dy = inputs(m, k, dtype=torch.bfloat16, seed=1), inputs(n, k, dtype=torch.bfloat16, seed=2, std=0.1), inputs(m, n, dtype=torch.bfloat16, seed=3)
    for compress in (True, False):
        check_linear(x, w, None, None, None, dy, compress)
        check_linear(x, w, None, "silu", None, dy, compress, (False, True, False))
        check_linear(x, w, None, None, None, dy, compress, (True, False, False))


@gpu
def test_linear_strides_and_shapes():
    dt = torch.bfloat16
    big = inputs(90, 500, dtype=dt, seed=1)
    wbig = inputs(400, 500, dtype=dt, seed=2, std=0.1)
    for x, w in ((big[:, 3:203], wbig[:70, :200]), (big[::2, 8:208], wbig[:64, 100:300]), (big[:, :64], wbig.t()[:72, :64]), (big.t()[:100], wbig[:33, :90]),
                 (big[:1].expand(70, 500), wbig), (big.view(9, 10, 500).transpose(0, 1), wbig[::2]), (big.view(3, 3, 10, 500)[:, :, 1:4], wbig[1:9])):
        n = w.shape[0]
        shape = x.shape[:-1] + (n,)
        dy = inputs(*shape, dtype=dt, seed=5, std=0.1)
        res = inputs(1, dtype=dt, seed=6).expand(shape)
        b = inputs(n + 1, dtype=dt, seed=7)[1:]
        for compress in (True, False):
            check_linear(x, w, b, "gelu", res, dy, compress)
            check_linear(x, w, b, None, None, dy[..., :1].expand(shape), compress)


@gpu
def test_linear_without_rows_and_without_saving():
    from gact import fused
    dt = torch.float16
    w, b = inputs(40, 24, dtype=dt, seed=1), inputs(40, dtype=dt, seed=2)
    for act in (None, "gelu"):
        for compress in (True, False):
            y, saved = fused.op_linear(torch.empty(3, 0, 24, dtype=dt, device="cuda"), w, b, act, compress=compress)
            dx, dw, db = fused.op_linear_backward(y, saved)
            assert y.shape == (3, 0, 40) and dx.shape == (3, 0, 24) and bool((dw == 0).all()) and bool((db == 0).all())
    x = inputs(10, 24, dtype=dt, seed=3)
    y, saved = fused.op_linear(x, w, b, "gelu", save=False)
    assert saved is None and torch.equal(y, fused.op_linear(x, w, b, "gelu")[0])


@gpu
def test_linear_shares_a_checkpoint():
    from gact import fused
    dt = torch.bfloat16
    x, w = inputs(50, 64, dtype=dt, seed=1), inputs(48, 64, dtype=dt, seed=2, std=0.1)
    c = fused.op_checkpoint8(x)
    check_linear(x, w, None, None, None, inputs(50, 48, dtype=dt, seed=3), True, checkpoint=c)
    assert fused.op_linear(x, w, checkpoint=c)[1].x is c


@gpu
def test_linear_keeps_special_values_in_their_rows():
    """A NaN or an infinity of x reaches its row of y and dW, and nothing else; values past the type's range become inf."""
    from gact import fused
    dt = torch.float16
    x, w = inputs(70, 64, dtype=dt, seed=1), inputs(40, 64, dtype=dt, seed=2, std=0.1)
    x[3, 5], x[64, 40] = float("nan"), float("inf")
    y, saved = fused.op_linear(x, w, None, "gelu")
    keep = torch.ones(70, dtype=torch.bool, device="cuda")
    keep[[3, 64]] = False
    assert y[keep].isfinite().all() and y[3].isnan().all() and not y[64].isfinite().all()
    dx, dw, _ = fused.op_linear_backward(torch.ones_like(y), saved)
    assert dx[keep].isfinite().all() and dw.isnan().any()
    big = torch.full((4, 64), 200.0, dtype=dt, device="cuda")
    assert bool((fused.op_linear(big, big)[0] == float("inf")).all())
