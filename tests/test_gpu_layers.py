"""gact.layers on a GPU: gradients against autograd in 64 bits, runs of several layers together, autocast, graphs, streams,
and a model that mixes them with a Controller's hooks."""
import math

import pytest
import torch
import torch.nn as nn

gpu = pytest.mark.gpu


def rand(*shape, seed=0, dtype=torch.bfloat16, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").mul_(std).to(dtype)


def rel(a, b):
    a, b = a.double(), b.double()
    return float((a - b).norm() / b.norm())


class Block(nn.Module):
    """The feed-forward half of a transformer block: y = x + W2 gelu(W1 norm(x))."""

    def __init__(self, width, inner, fused):
        super().__init__()
        from gact import layers
        self.fused = fused
        if fused:
            self.norm, self.up, self.down = layers.LayerNorm(width), layers.Linear(width, inner, activation="gelu"), layers.Linear(inner, width)
        else:
            self.norm, self.up, self.down = nn.LayerNorm(width), nn.Linear(width, inner), nn.Linear(inner, width)

    def forward(self, x):
        if self.fused:
            return self.down(self.up(self.norm(x)), residual=x)
        return x + self.down(nn.functional.gelu(self.up(self.norm(x))))


def blocks(width, inner, n, dtype):
    """n blocks on gact.layers, and the same parameters in 64 bits on torch's layers."""
    torch.manual_seed(5)
    ref = nn.Sequential(*[Block(width, inner, False) for _ in range(n)]).cuda().to(dtype)
    own = nn.Sequential(*[Block(width, inner, True) for _ in range(n)]).cuda().to(dtype)
    own.load_state_dict(ref.state_dict())
    return own, ref.double()


@gpu
@pytest.mark.parametrize("compress", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_blocks_against_autograd_in_64_bits(dtype, compress):
    """Three blocks in a row, as they are used.  Each stored activation is off by at most half a step of its type, each
    gradient too: about 10 roundings lie between the input and the first block's gradients, 3 more (the checkpoints of norm
    input, linear input and pre-activation) with a relative size of at most 2^-7 of the largest in 32 each."""
    import gact
    gact.config.compress_activation = compress
    own, ref = blocks(96, 200, 3, dtype)
    x = rand(70, 96, seed=1, dtype=dtype).requires_grad_()
    x64 = x.detach().double().requires_grad_()
    dy = rand(70, 96, seed=2, dtype=dtype, std=0.1)
    y, y64 = own(x), ref(x64)
    half = torch.finfo(dtype).eps / 2
    assert rel(y, y64) < 12 * half
    y.backward(dy)
    y64.backward(dy.double())
    # a code is off by at most half a step and a step is at most 2^-6.0 of the largest of its 32; relative to the typical
    # value (a third of the largest) that is 3 * 2^-7 at most, in each of 3 places per block
    bound = 30 * half + (9 * 3 * 2.0 ** -7 if compress else 0)
    assert rel(x.grad, x64.grad) < bound
    for (name, p), q in zip(own.named_parameters(), ref.parameters()):
        assert rel(p.grad, q.grad) < bound, name


@gpu
def test_gradients_against_differences():
    """Directional derivatives of a linear + layer norm in 64-bit differences of the plain formula."""
    from gact import layers
    import gact
    gact.config.compress_activation = False
    dt = torch.float16
    x, w = rand(40, 64, seed=1, dtype=dt), rand(48, 64, seed=2, dtype=dt, std=0.15)
    b, g, h = rand(48, seed=3, dtype=dt), rand(48, seed=4, dtype=dt) + 1, rand(48, seed=5, dtype=dt)
    dy = rand(40, 48, seed=6, dtype=dt, std=0.1)
    leaves = [t.clone().requires_grad_() for t in (x, w, b, g, h)]
    y = layers.layer_norm(layers.linear(leaves[0], leaves[1], leaves[2], "silu"), leaves[3], leaves[4])
    y.backward(dy)

    def f(x, w, b, g, h):
        z = nn.functional.silu(x @ w.t() + b)
        return (nn.functional.layer_norm(z, (48,), g, h) * dy.double()).sum()

    base = [t.double() for t in (x, w, b, g, h)]
    for i, leaf in enumerate(leaves):
        d = rand(*leaf.shape, seed=20 + i, dtype=torch.float64)
        e = 1e-6
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + e * d, base[i] - e * d
        diff = float((f(*up) - f(*down)) / (2 * e))
        got = float((leaf.grad.double() * d).sum())
        # roundings of y, dz and the gradient itself: a few half steps (2^-11) of the sum of magnitudes over the root of n
        tol = 8 * 2.0 ** -11 * float((leaf.grad.double() * d).abs().sum()) / math.sqrt(leaf.numel()) + 8 * 2.0 ** -11 * abs(diff)
        assert abs(got - diff) < tol + 8 * 2.0 ** -11 * float(leaf.grad.double().norm()), i


@gpu
def test_autocast_casts_like_torch_and_returns_gradients_in_the_parameters_type():
    from gact import layers
    m = layers.Linear(64, 32, activation="relu").cuda()
    n = layers.LayerNorm(32).cuda()
    x = rand(10, 64, dtype=torch.float32).requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = m(x)
        z = n(y)
    assert y.dtype == z.dtype == torch.bfloat16
    z.float().square().sum().backward()
    assert x.grad.dtype == m.weight.grad.dtype == m.bias.grad.dtype == n.weight.grad.dtype == torch.float32
    assert all(torch.isfinite(t).all() for t in (x.grad, m.weight.grad, m.bias.grad, n.weight.grad))
    assert n(x.detach()[:, :32]).dtype == torch.float32
    with pytest.raises(RuntimeError, match="autocast"):
        m(x)


@gpu
def test_what_is_kept_and_that_hooks_leave_it_alone():
    """Under a Controller the layers' int8 codes, statistics and parameters pass the hooks untouched, other saves are
    compressed, and the gradients are those of the layers without hooks."""
    import gact
    from gact import layers
    gact.set_optimization_level("L1")

    def run(hooks):
        torch.manual_seed(0)
        m = nn.Sequential(layers.Linear(64, 128, activation="gelu"), layers.LayerNorm(128), layers.Linear(128, 64)).cuda().bfloat16()
        c = gact.Controller(m)
        x = rand(50, 64, seed=1)
        if hooks:
            c.install_hook()
        y = m(x)
        out = y.float().square().sum()
        n = c.quantizer.tid
        out.backward()
        if hooks:
            c.uninstall_hook()
        return [p.grad for p in m.parameters()], n

    plain, _ = run(False)
    hooked, n = run(True)
    assert n == 1                                   # y.float().square() saves one activation, the layers none
    # that one is the only difference: 4 bits of y.float()
    for a, b in zip(plain, hooked):
        assert rel(b, a) < 0.2
    y = layers.linear(rand(64, 64, seed=2).requires_grad_(), rand(32, 64, seed=3), None, "gelu")
    kept = y.grad_fn.saved_tensors
    assert all(t is None or t.dtype in (torch.int8, torch.bfloat16) for t in kept) and kept[0].dtype == torch.int8


@gpu
def test_memory_of_a_block_is_the_codes():
    from gact import layers
    x = rand(4096, 1024).requires_grad_()
    w1, w2 = rand(4096, 1024, std=0.03).requires_grad_(), rand(1024, 4096, std=0.03).requires_grad_()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = layers.linear(layers.linear(x, w1, None, "gelu"), w2)
    torch.cuda.synchronize()
    kept = torch.cuda.memory_allocated() - before - y.numel() * 2
    codes = 4096 * (1024 + 4096 + 4096) * 33 // 32
    assert codes <= kept < codes + (1 << 20)


@gpu
def test_convert_and_sequential_activation():
    from gact import layers
    torch.manual_seed(1)
    m = nn.Sequential(nn.Linear(64, 128), nn.GELU(approximate="tanh"), nn.LayerNorm(128), nn.Linear(128, 8), nn.Tanh()).cuda().half()
    x = rand(33, 64, dtype=torch.float16)
    want = m(x)
    out = layers.convert(m)
    assert out is m and type(m[0]) is layers.Linear and m[0].activation == "gelu_tanh" and type(m[1]) is nn.Identity
    assert type(m[2]) is layers.LayerNorm and type(m[3]) is layers.Linear and type(m[4]) is nn.Tanh
    assert rel(m(x), want) < 0.01
    n = layers.LayerNorm((4, 16)).cuda()
    y = torch.randn(3, 4, 16, device="cuda")
    assert torch.allclose(n(y), nn.functional.layer_norm(y, (4, 16)), atol=1e-5)


@gpu
def test_share_input_gives_the_same_gradients_with_one_checkpoint():
    from gact import layers

    class Three(nn.Module):
        def __init__(self):
            super().__init__()
            self.a, self.b, self.c = (layers.Linear(64, 64) for _ in range(3))

        def forward(self, x):
            return self.a(x) * self.b(x) + self.c(x)

    torch.manual_seed(0)
    m = Three().cuda().bfloat16()
    x = rand(256, 64, seed=1).requires_grad_()
    m(x).float().square().sum().backward()
    want = [p.grad.clone() for p in m.parameters()] + [x.grad.clone()]
    m.zero_grad(), setattr(x, "grad", None)
    layers.share_input(m, (m.a, m.b, m.c))
    y = m(x)
    assert m.a._shared is None
    y.float().square().sum().backward()
    for a, b in zip([p.grad for p in m.parameters()] + [x.grad], want):
        assert torch.equal(a, b)
    with torch.no_grad():
        m(x)
    m(x.detach())


@gpu
def test_a_training_step_in_a_graph_next_to_an_eager_one():
    """Forward and backward captured on their own leaves; replays follow new inputs, and an eager step of other leaves runs
    between them without disturbing either."""
    from gact import layers
    own, _ = blocks(64, 128, 2, torch.bfloat16)
    params = list(own.parameters())
    x = rand(40, 64, seed=1)
    dy = rand(40, 64, seed=2, std=0.1)

    def step():
        y = own(x)
        return [y] + list(torch.autograd.grad(y, params, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    other, _ = blocks(64, 128, 1, torch.bfloat16)
    for seed in (3, 4):
        x.copy_(rand(40, 64, seed=seed))
        g.replay()
        got = [t.clone() for t in out]
        other(rand(30, 64, seed=seed)).float().sum().backward()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


@gpu
def test_two_streams_at_once_give_the_results_of_one():
    from gact import fused
    cases = []
    for i in range(2):
        x, w = rand(512, 256, seed=i), rand(320, 256, seed=10 + i, std=0.1)
        cases.append((x, w, rand(320, seed=20 + i), rand(512, 320, seed=30 + i), rand(512, 256, seed=40 + i, dtype=torch.float32)))

    def work(c):
        x, w, b, dy, n = c
        y, s = fused.op_linear(x, w, b, "gelu")
        z, t = fused.op_layer_norm(n)
        return [y, z, *fused.op_linear_backward(dy, s), fused.op_layer_norm_backward(n, t)[0]]

    want = [work(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(work(c))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            for a, b in zip(g, w):
                assert torch.equal(a, b)


@gpu
def test_results_do_not_vary_from_run_to_run():
    from gact import fused
    x, w, b = rand(3000, 520, seed=1), rand(264, 520, seed=2, std=0.1), rand(264, seed=3)
    dy = rand(3000, 264, seed=4)

    def all_():
        y, s = fused.op_linear(x, w, b, "gelu")
        n, t = fused.op_layer_norm(x, w[0], w[1])
        return [y, n, *fused.op_linear_backward(dy, s), *fused.op_layer_norm_backward(x, t)]

    first = all_()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, all_()))


@gpu
def test_stochastic_checkpoints_follow_the_config():
    import gact
    from gact import layers
    x, w = rand(64, 64, seed=1).requires_grad_(), rand(64, 64, seed=2)
    for stochastic in (True, False):
        gact.config.stochastic_checkpoints = stochastic
        y, z = layers.linear(x, w), layers.linear(x, w)
        assert torch.equal(y.grad_fn.saved_tensors[0], z.grad_fn.saved_tensors[0]) is not stochastic


@gpu
def test_bert_workload_on_fused_layers():
    """Two BERT-large layers through the training driver: a step and an adaptation run at L1 and L2, gradients are finite and
    near those of torch's layers (same weights, no dropout, no compression elsewhere)."""
    import gact
    import workloads
    dev = torch.device("cuda", 0)
    gact.set_optimization_level("L0")

    def grads(fused):
        wl = workloads.bert_large(dev, batch=4, layers=2, fused=fused)
        for m in wl.model.modules():
            if isinstance(m, nn.Dropout):
                m.p = 0.0
        wl.model.config.attention_probs_dropout_prob = 0.0
        for b in wl.model.bert.encoder.layer:
            if hasattr(b.attention.self, "dropout") and isinstance(b.attention.self.dropout, nn.Dropout):
                b.attention.self.dropout.p = 0.0
        loss, _ = wl.forward()
        loss.backward()
        return float(loss), {n: p.grad.clone() for n, p in wl.model.named_parameters()}

    l0, want = grads(False)
    gact.config.compress_activation = True          # the fused layers keep codes, no hooks installed
    l1, got = grads(True)
    assert abs(l0 - l1) < 0.05 and want.keys() == got.keys()
    a = torch.cat([want[n].flatten() for n in want]).double()
    b = torch.cat([got[n].flatten() for n in want]).double()
    assert torch.isfinite(b).all() and float((a - b).norm() / a.norm()) < 0.2
    for level in ("L1", "L2"):
        gact.config.reset()
        gact.set_optimization_level(level)
        wl = workloads.bert_large(dev, batch=8, layers=2, fused=True)
        c = gact.Controller(wl.model)
        c.install_hook()
        for _ in range(2):
            loss = wl.step()
            c.iterate(wl.backprop)
        c.uninstall_hook()
        assert torch.isfinite(loss)
        assert all(torch.isfinite(p).all() for p in wl.model.parameters())


@gpu
def test_share_input_notices_another_tensor():
    """A child that is given something else than the parent's argument (here: the argument changed in place, and a sum) keeps its
    own checkpoint."""
    from gact import layers

    class Other(nn.Module):
        def __init__(self):
            super().__init__()
            self.a, self.b = layers.Linear(64, 64), layers.Linear(64, 64)

        def forward(self, x):
            return self.a(x + 1) + self.b(x)

    torch.manual_seed(0)
    m = Other().cuda().bfloat16()
    x = rand(32, 64, seed=1)
    grads = []
    for share in (False, True):
        if share:
            layers.share_input(m, (m.a, m.b))
        m.zero_grad()
        m(x).float().square().sum().backward()
        grads.append([p.grad.clone() for p in m.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*grads))


@gpu
def test_second_derivatives_are_refused_and_kept_graphs_work():
    from gact import layers
    x, w = rand(16, 32, seed=1).requires_grad_(), rand(8, 32, seed=2).requires_grad_()
    y = layers.layer_norm(layers.linear(x, w, None, "gelu"))
    a = torch.autograd.grad(y.float().square().sum(), [x, w], retain_graph=True)
    b = torch.autograd.grad(y.float().square().sum(), [x, w])
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    y = layers.linear(x, w)
    (g,) = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
