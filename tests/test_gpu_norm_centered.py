"""Layer norm's centred checkpoints: rows whose mean is large against their deviation, where codes of the input itself fail.

Tolerances are bounds, worked out before the first run.  With d = x - mean: the kernel's mean is a sum of at most 24 additions one
after the other and a product, so it is off by e = 28 * 2^-24 * mean|x|.  A code is off by half a step and a step is at most 1/63.5 of
its block's largest magnitude, so a kept value is off by E = (max|d| + e) / 127 + e, and x^ by E r.  The variance is off by
2 e rms(d) + e^2, which moves r by half of that relative to var + eps.
"""
import pytest
import torch

gpu = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U24 = 2.0 ** -24


def rand(*shape, seed=0, std=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").mul_(std).to(dtype)


def within(got, want, tol, what):
    got, want, tol = got.detach().double().cpu(), want.cpu(), tol.cpu()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), "%s: %d of %d off, worst by %g" % (what, int(bad.sum()), bad.numel(), float(((got - want).abs() - tol).max()))


def check(x, w, b, dy, eps=1e-5, seed=None):
    from gact import fused
    y, saved = fused.op_layer_norm(x, w, b, eps, seed=seed, center=True)
    dx, dw, db = fused.op_layer_norm_backward(dy, saved)
    plain = fused.op_layer_norm(x, w, b, eps, compress=False)
    assert torch.equal(y, plain[0]) and torch.equal(saved.stats[:, 1], plain[1].stats[:, 1]) and not saved.stats[:, 0].any()
    x, w, dy = x.double().cpu(), w.double().cpu(), dy.double().cpu()
    rows = x.shape[0]
    mean = x.mean(1, keepdim=True)
    d = x - mean
    var = (d * d).mean(1, keepdim=True)
    r = (var + eps).rsqrt()
    e = 28 * U24 * x.abs().mean(1, keepdim=True)
    top = d.abs().amax(1, keepdim=True)
    E = (top + e) / 127 * (1 if seed is None else 2) + e
    kept = fused.op_restore8(saved.x)
    assert kept.dtype == torch.float32
    within(kept, d, (E + U24 * d.abs()).expand_as(d), "kept")
    xh = d * r
    dr = 0.5 * (2 * e * var.sqrt() + e * e) / (var + eps) + 8 * U24
    xe = r * (1 + dr) * E + xh.abs() * (dr + 4 * U24)
    g = dy * w
    c1, c2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    c2e = (g.abs() * xe).mean(1, keepdim=True) + 64 * U24 * (g * xh).abs().mean(1, keepdim=True)
    inner = 8 * U24 * (g.abs() + c1.abs() + (xh * c2).abs()) + 64 * U24 * g.abs().mean(1, keepdim=True) + xe * (c2.abs() + c2e) + xh.abs() * c2e
    want = r * (g - c1 - xh * c2)
    h = torch.finfo(dx.dtype).eps / 2 * 1.01
    tiny = torch.finfo(dx.dtype).tiny
    within(dx, want, h * want.abs() + (1 + h) * (r * (1 + dr) * inner + dr * want.abs()) + tiny, "dx")
    hp = torch.finfo(dw.dtype).eps / 2 * 1.01
    k = (64 + rows / 64) * U24
    want = (dy * xh).sum(0)
    within(dw, want, hp * want.abs() + (1 + hp) * ((dy.abs() * xe).sum(0) + k * (dy * xh).abs().sum(0)) + torch.finfo(dw.dtype).tiny, "dw")
    within(db, dy.sum(0), hp * dy.sum(0).abs() + 1.01 * k * dy.abs().sum(0) + torch.finfo(db.dtype).tiny, "db")


# row lengths of every kernel shape, with and without rows on 16-byte boundaries, one block and a short last block
@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 33), (40, 64), (9, 100), (2000, 96), (2000, 256), (33, 257), (2000, 512), (2000, 1024), (70, 771), (1300, 2048),
                                       (21, 1500), (1300, 4096), (7, 5001), (1300, 8192), (3, 16384)])
@pytest.mark.parametrize("mean", [0.0, 100.0])
def test_centered_layer_norm(rows, cols, dtype, mean):
    dt = DT[dtype]
    x = (rand(rows, cols, seed=1) + mean).to(dt)
    w, b = rand(cols, seed=2, std=0.2, dtype=dt) + 1, rand(cols, seed=3, dtype=dt)
    check(x, w, b, rand(rows, cols, seed=4, std=0.1, dtype=dt))


@gpu
def test_centered_rows_that_hardly_vary():
    """Rows of 100.3 +- 0.01, constant rows that no code holds (1.01), constant rows of 16-bit types, fp32 weights."""
    x = rand(50, 1000, seed=1, std=0.01) + 100.3
    x[3], x[7] = 1.01, -77.7
    w, b, dy = rand(1000, seed=2, std=0.2) + 1, rand(1000, seed=3), rand(50, 1000, seed=4)
    check(x, w, b, dy)
    check(x.bfloat16(), w, b, dy.bfloat16())
    check(x[:, :-1], w[1:], b[1:], dy[:, 1:])
    from gact import fused
    c = torch.full((4, 1024), 1.01, device="cuda")
    _, saved = fused.op_layer_norm(c, center=True)
    dy = rand(4, 1024, seed=5)
    dx = fused.op_layer_norm_backward(dy, saved)[0]
    # nothing but the centring of dy is left: r (g - mean(g)) with r = 1 / sqrt(eps)
    want = (dy - dy.mean(1, keepdim=True)).double() / 1e-5 ** 0.5
    assert float((dx.double() - want).norm() / want.norm()) < 1e-3


@gpu
def test_centered_values_beyond_the_range_of_fp16():
    x = torch.full((3, 64), 65504.0, device="cuda", dtype=torch.float16)
    x[:, 5] = -65504.0
    x[1, 6:40] = -65000.0
    check(x, torch.ones(64, device="cuda", dtype=torch.float16), torch.zeros(64, device="cuda", dtype=torch.float16), rand(3, 64, seed=1, dtype=torch.float16))


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_centered_stochastic_codes(dtype):
    from gact import fused
    x = (rand(300, 200, seed=1) + 30).to(DT[dtype])
    w, b, dy = rand(200, seed=2) + 1, rand(200, seed=3), rand(300, 200, seed=4, dtype=DT[dtype])
    check(x, w, b, dy, seed=9)
    a, c = (fused.op_layer_norm(x, seed=s, center=True)[1].x.buf for s in (9, 10))
    assert not torch.equal(a, c) and torch.equal(a, fused.op_layer_norm(x, seed=9, center=True)[1].x.buf)


@gpu
def test_centered_special_rows():
    """A NaN or an infinity stays in its row; no rows, one element."""
    from gact import fused
    x = rand(6, 96, seed=1, dtype=torch.bfloat16)
    x[2, 5], x[3, 70] = float("nan"), float("inf")
    w, b = rand(96, seed=2, dtype=torch.bfloat16), rand(96, seed=3, dtype=torch.bfloat16)
    y, saved = fused.op_layer_norm(x, w, b, center=True)
    dx, dw, db = fused.op_layer_norm_backward(torch.ones_like(x), saved)
    good = [0, 1, 4, 5]
    assert y[good].isfinite().all() and dx[good].isfinite().all()
    assert y[2].isnan().all() and y[3].isnan().all() and dx[2].isnan().all() and dx[3].isnan().all() and bool((db == 6).all())
    y, saved = fused.op_layer_norm(x[:0], w, b, center=True)
    dx, dw, db = fused.op_layer_norm_backward(y, saved)
    assert dx.shape == (0, 96) and not dw.any() and not db.any()
    y, saved = fused.op_layer_norm(x, w, b, save=False, center=True)
    assert saved is None


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_layers_keep_their_gradients_where_the_mean_is_large(dtype):
    """Modules and the function, mean 100 times the deviation: a code's error is uniform in half a step of at most 1/63.5 of the block's
    largest (up to 4 deviations), so x^ and with it dw are off by at most 4 / 63.5 / sqrt(12) = 1.8 % in the root mean square; 2^-8 for
    each of the roundings of x, dx and dw in bf16."""
    from gact import layers
    dt = DT[dtype]
    x = (rand(500, 1024, seed=1) + 100).to(dt).requires_grad_()
    dy = rand(500, 1024, seed=2, dtype=dt)
    m = layers.LayerNorm(1024).cuda().to(dt)
    m(x).backward(dy)
    x64 = x.detach().double().requires_grad_()
    n = torch.nn.LayerNorm(1024).cuda().double()
    n(x64).backward(dy.double())
    for got, want in ((x.grad, x64.grad), (m.weight.grad, n.weight.grad), (m.bias.grad, n.bias.grad)):
        assert float((got.double() - want).norm() / want.norm()) < 0.018 + 3 * 2.0 ** -8
