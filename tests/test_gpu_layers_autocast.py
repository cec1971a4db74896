"""gact.layers under autocast next to tensors of other types."""
import pytest
import torch

gpu = pytest.mark.gpu


def rand(*shape, seed=0, dtype=torch.float32, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").mul_(std).to(dtype)


@gpu
@pytest.mark.parametrize("act", [None, "gelu"])
def test_an_fp32_residual_keeps_its_bits(act):
    from gact import layers
    m = layers.Linear(64, 32, activation=act).cuda()
    x, r = rand(40, 64, seed=1).requires_grad_(), (rand(40, 32, seed=2) + 1000).requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = m(x, residual=r)
        z = m(x)
        narrow = m(x, residual=r.detach().bfloat16())
        with pytest.raises(ValueError, match="residual"):
            m(x, residual=r[0])
    assert y.dtype == torch.float32 and torch.equal(y, z.float() + r) and narrow.dtype == torch.bfloat16
    dy = rand(40, 32, seed=3)
    y.backward(dy)
    assert torch.equal(r.grad, dy)
    got = m.weight.grad.clone()
    m.zero_grad()
    z.backward(dy.bfloat16())
    assert torch.equal(got, m.weight.grad)
    with pytest.raises(RuntimeError, match="residual"):
        layers.linear(rand(40, 64, dtype=torch.bfloat16), rand(32, 64, dtype=torch.bfloat16), residual=r)
