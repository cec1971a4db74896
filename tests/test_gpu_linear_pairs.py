"""Products on pairs of blocks, launched back to back with kernels that keep their own barriers in the same SMs' shared memory."""
import pytest
import torch

gpu = pytest.mark.gpu


def rand(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").bfloat16()


@gpu
def test_pairs_leave_nothing_behind_for_the_next_kernel():
    """A block of a pair ends only after the last arrival that the other one sends to its shared memory: 400 launches of short
    pair products, each followed by layer norm's rings and a single-block product on the same SMs, repeat their results."""
    from gact import _native as nv, fused
    x, w = rand(2048, 1024, seed=1), rand(2048, 1024, seed=2)
    n, small = rand(1500, 2048, seed=3), rand(64, 256, seed=4)
    _, kept = fused.op_layer_norm(n)
    first = None
    for i in range(400):
        got = [fused.op_linear(x, w, save=False)[0], fused.op_layer_norm_backward(n, kept)[0], fused.op_linear(small, small, save=False)[0]]
        if first is None:
            first = got
        elif i % 40 == 0:
            assert all(torch.equal(a, b) for a, b in zip(first, got))
    assert all(torch.equal(a, b) for a, b in zip(first, got))
    assert nv.lib.gact_pipeline_error() == 0
