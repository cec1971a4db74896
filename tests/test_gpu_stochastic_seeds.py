"""Seeds of stochastic checkpoints that lie on the device, and captured steps whose replays draw new noise."""
import gc
import math

import pytest
import torch

gpu = pytest.mark.gpu


def rand(*shape, seed=0, dtype=torch.bfloat16, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").mul_(std).to(dtype)


def word(v):
    return torch.tensor([v], dtype=torch.int64, device="cuda")


def philox7(counter, high):
    """Philox4x32 with 7 rounds and key 0 on Python integers."""
    c = [counter & 0xffffffff, counter >> 32, high & 0xffffffff, high >> 32]
    k0 = k1 = 0
    for _ in range(7):
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(p1 >> 32) ^ c[1] ^ k0, p1 & 0xffffffff, (p0 >> 32) ^ c[3] ^ k1, p0 & 0xffffffff]
        k0, k1 = (k0 + 0x9E3779B9) & 0xffffffff, (k1 + 0xBB67AE85) & 0xffffffff
    return c


@gpu
def test_codes_of_a_device_seed_match_the_generator():
    from gact import fused
    x, seed = rand(5, 71, dtype=torch.float32, seed=11), 0x123456789ABCDEF
    c = fused.op_checkpoint8(x, word(seed))
    codes, scales, xs = c.codes.cpu(), c.scales.cpu().view(torch.uint8), x.cpu().double()
    for r in range(5):
        for col in range(71):
            i = r * 96 + col
            w = philox7(i // 8, seed)[(i % 8) // 2]
            u = (((w >> 16) if i & 1 else (w & 0xffff)) + 0.5) / 65536
            v = float(xs[r, col]) * 2.0 ** (127 - int(scales[r, col // 32]))
            assert int(codes[r, col]) in (math.floor(v + u), math.floor(float(torch.tensor(v + u, dtype=torch.float32)))), (r, col)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(3, 33), (300, 200), (50, 1003), (4000, 1024), (2000, 2056)])
def test_device_seeds_repeat_and_differ(rows, cols, dtype):
    """The same value gives the same codes wherever they are made, another value others; a code is within a step of its value."""
    from gact import fused
    x = rand(rows, cols, seed=1, dtype=dtype)
    a = fused.op_checkpoint8(x, word(7))
    assert torch.equal(a.buf, fused.op_checkpoint8(x, word(7)).buf) and not torch.equal(a.buf, fused.op_checkpoint8(x, word(8)).buf)
    assert not torch.equal(a.buf, fused.op_checkpoint8(x, 7).buf) and torch.equal(a.scales, fused.op_checkpoint8(x).scales)
    assert torch.equal(a.buf, fused.op_layer_norm(x, seed=word(7))[1].x.buf)
    assert not torch.equal(fused.op_layer_norm(x, seed=word(7), center=True)[1].x.buf, fused.op_layer_norm(x, seed=word(8), center=True)[1].x.buf)
    # the value 0 on the device is the key 0 and a counter of 0 above: a plain seed of 0
    assert torch.equal(fused.op_checkpoint8(x, word(0)).buf, fused.op_checkpoint8(x, 0).buf)
    step = torch.exp2(a.scales.view(torch.uint8).double() - 127).repeat_interleave(32, 1)[:, :cols]
    assert bool(((fused.op_restore8(a, torch.float32).double() - x.double()).abs() <= step * (1 + 2.0 ** -16)).all())
    if dtype is not torch.float32:
        w = rand(40, cols, seed=2, dtype=dtype, std=0.05)
        for act in ("gelu", "relu"):
            s, t, u = (fused.op_linear(x, w, None, act, seed=word(v))[1] for v in (7, 7, 8))
            assert torch.equal(s.x.buf, a.buf) and torch.equal(s.z.buf, t.z.buf) and not torch.equal(s.z.buf, u.z.buf)


@gpu
def test_seed_refusals():
    from gact import fused
    x, w = rand(4, 16), rand(8, 16)
    for call in (lambda s: fused.op_checkpoint8(x, s), lambda s: fused.op_layer_norm(x, seed=s), lambda s: fused.op_linear(x, w, seed=s)):
        for seed, error in ((torch.tensor([1]), RuntimeError), (word(1).int(), ValueError), (word(1).repeat(2), ValueError), (word(1).double(), ValueError),
                            ("1", TypeError), (1.5, TypeError)):
            with pytest.raises(error):
                call(seed)


@gpu
def test_replays_of_a_captured_step_draw_new_noise():
    """Linear (shared input, epilogue) and layer norm with stochastic checkpoints, captured: replays on the same inputs give other
    weight gradients, and their mean approaches that of the step without compression."""
    import gact
    from gact import layers

    class Pair(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.norm, self.a, self.b = layers.LayerNorm(64), layers.Linear(64, 32), layers.Linear(64, 32, activation="silu")

        def forward(self, x):
            return self.a(x) + self.b(x) + self.norm(x)[..., :32]

    torch.manual_seed(0)
    m = Pair().cuda().bfloat16()
    layers.share_input(m, (m.a, m.b))
    x, dy = rand(200, 64, seed=1), rand(200, 32, seed=2, std=0.1)
    params = list(m.parameters())

    def step():
        return torch.autograd.grad(m(x), params, dy)

    gact.config.compress_activation = False
    exact = [g.double() for g in step()]
    gact.config.compress_activation = True
    gact.config.stochastic_checkpoints = True
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    gc.collect()                                   # (no graph of another test may be collected inside the capture)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    n = 200
    first, total = None, [torch.zeros_like(e) for e in exact]
    for i in range(n):
        g.replay()
        for t, o in zip(total, out):
            t += o.double()
        if i == 0:
            first = [o.clone() for o in out]
        elif i == 1:
            names = [k for k, _ in m.named_parameters()]
            differ = {k for k, a, b in zip(names, first, out) if not torch.equal(a, b)}
            assert differ >= {"norm.weight", "a.weight", "b.weight"}
    # One gradient's error is the sum of 200 rounding errors of variance below (step / 2)^2; a step is at most 1/63.5 of the largest (under 4
    # deviations) of 32, so it is below 4 / 63.5 / 2 = 3.2 % of the typical product.  The mean of n keeps 1 / sqrt(n) of that, beside
    # the 16-bit roundings of the stored values (2^-8 each for the output and dz; the silu layer's slope of a rounded z adds a bias of
    # the order of its square, 0.1 %).
    for t, e in zip(total, exact):
        assert float((t / n - e).norm() / e.norm()) < 3 * 0.032 / math.sqrt(n) + 2 * 2.0 ** -8 + 0.001
