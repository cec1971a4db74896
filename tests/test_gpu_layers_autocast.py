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


@gpu
@pytest.mark.parametrize("x,w,b", [("float32", "bfloat16", "bfloat16"), ("float32", "float16", None), ("bfloat16", "float16", "float16"),
                                   ("bfloat16", "bfloat16", "float32"), ("float16", None, "bfloat16")])
def test_layer_norm_under_autocast_takes_parameters_of_other_types(x, w, b):
    """As torch does, which widens everything; without autocast they are an error, as torch's are."""
    from gact import layers
    t = lambda name, *shape, seed: None if name is None else rand(*shape, seed=seed, dtype=getattr(torch, name)).requires_grad_()
    x, w, b = t(x, 30, 96, seed=1), t(w, 96, seed=2), t(b, 96, seed=3)
    with pytest.raises(RuntimeError, match="type"):
        layers.layer_norm(x, w, b)
    dy = rand(30, 96, seed=4)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = layers.layer_norm(x, w, b, compress=False)
        want = torch.nn.functional.layer_norm(x, (96,), w, b)
    leaves = [p for p in (x, w, b) if p is not None]
    got = torch.autograd.grad(y, leaves, dy.to(y.dtype))
    ref = torch.autograd.grad(want, leaves, dy.to(y.dtype).float())
    half = torch.finfo(x.dtype).eps / 2
    # y and each gradient are stored once in their own type; 64 steps of fp32 for the sums
    assert y.dtype == x.dtype and float((y.detach().double() - want.detach().double()).norm() / want.detach().double().norm()) < half + 64 * 2.0 ** -24
    for p, g, r in zip(leaves, got, ref):
        e = torch.finfo(p.dtype).eps
        assert g.dtype == p.dtype and float((g.double() - r.double()).norm() / r.double().norm()) < e + 64 * 2.0 ** -24
