"""gact.layers next to a Controller's hooks, under autocast."""
import pytest
import torch
import torch.nn as nn

gpu = pytest.mark.gpu


def rand(*shape, seed=0, dtype=torch.float32, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").mul_(std).to(dtype)


@gpu
@pytest.mark.parametrize("native", [True, False])
def test_hooks_leave_the_weights_alone_under_autocast(native):
    """fp32 parameters, autocast, a Controller: the layers' saves take no number of the quantizer, and with nothing else to
    compress every gradient is that of the step without hooks, bit for bit."""
    import gact
    from gact import layers
    gact.set_optimization_level("L1")
    gact.config.native_hooks = native

    def run(hooks):
        torch.manual_seed(0)
        m = nn.Sequential(layers.Linear(64, 128, activation="gelu"), layers.LayerNorm(128), layers.Linear(128, 64), layers.Linear(64, 32)).cuda()
        c = gact.Controller(m)
        x, dy = rand(50, 64, seed=1).requires_grad_(), rand(50, 32, seed=2, dtype=torch.bfloat16)
        if hooks:
            c.install_hook()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = m(x)
        n = c.quantizer.tid
        y.backward(dy)
        if hooks:
            c.uninstall_hook()
        assert y.dtype == torch.bfloat16 and all(p.grad.dtype == torch.float32 for p in m.parameters())
        return [x.grad] + [p.grad for p in m.parameters()], n

    plain, _ = run(False)
    hooked, n = run(True)
    assert n == 0
    assert all(torch.equal(a, b) for a, b in zip(plain, hooked))
