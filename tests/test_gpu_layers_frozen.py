"""Linear layers with frozen weights or inputs: what they keep, and that the gradients that are left stay the same."""
import pytest
import torch

gpu = pytest.mark.gpu


def rand(*shape, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").mul_(std).bfloat16()


@gpu
@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("compress", [True, False])
def test_gradients_that_are_left_stay_the_same(act, compress):
    from gact import layers
    data = rand(300, 200, seed=1), rand(120, 200, seed=2, std=0.1), rand(120, seed=3), rand(300, 120, seed=4)
    dy = rand(300, 120, seed=5)

    def grads(mask):
        leaves = [torch.nn.Parameter(t.clone(), requires_grad=g) for t, g in zip(data, mask)]
        y = layers.linear(leaves[0], leaves[1], leaves[2], act, leaves[3], compress=compress)
        y.backward(dy)
        return y.detach(), [t.grad for t in leaves]

    y, full = grads((True,) * 4)
    for mask in [(True, False, False, False), (False, True, False, False), (False, False, True, False), (False, False, False, True), (True, False, True, False),
                 (False, True, True, True), (True, False, True, True)]:
        z, got = grads(mask)
        assert torch.equal(y, z)
        for g, want, asked in zip(got, full, mask):
            assert (g is not None) == asked and (g is None or torch.equal(g, want))


@gpu
@pytest.mark.parametrize("compress", [True, False])
def test_memory_of_frozen_layers(compress):
    """With frozen weights two layers keep their pre-activation and nothing else, through autograd and under autocast."""
    from gact import layers
    x = rand(4096, 1024).requires_grad_()
    a, b = layers.Linear(1024, 4096, activation="gelu").cuda(), layers.Linear(4096, 1024).cuda()
    for m in (a, b):
        m.requires_grad_(False)
    import gact
    gact.config.compress_activation = compress
    with torch.autocast("cuda", dtype=torch.bfloat16):
        a(x), b(a(x).detach())
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = b(a(x))
    torch.cuda.synchronize()
    kept = torch.cuda.memory_allocated() - before - y.numel() * 2
    z = 4096 * 4096 * 33 // 32 if compress else 4096 * 4096 * 2
    assert z <= kept < z + (1 << 20)


@gpu
def test_gradients_nobody_prepared_for_are_refused():
    from gact import fused
    x, w = rand(40, 64), rand(32, 64, seed=1)
    c = fused.op_checkpoint8(x)
    for kw in ({}, {"compress": False}, {"checkpoint": c}):
        y, saved = fused.op_linear(x, w, None, "gelu", keep_input=False, **kw)
        assert saved.x is None
        want = fused.op_linear_backward(y, fused.op_linear(x, w, None, "gelu", **kw)[1])
        assert torch.equal(fused.op_linear_backward(y, saved, (True, False, False))[0], want[0])
        with pytest.raises(ValueError, match="not saved"):
            fused.op_linear_backward(y, saved)
        y, saved = fused.op_linear(x, w, **kw)
        saved.weight = None
        assert torch.equal(fused.op_linear_backward(y, saved, (False, True, False))[1], fused.op_linear_backward(y, fused.op_linear(x, w, **kw)[1])[1])
        with pytest.raises(ValueError, match="not saved"):
            fused.op_linear_backward(y, saved)
