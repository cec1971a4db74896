"""Bounded waits of the products and of layer norm's rings: the limit that is asked for, and who learns of a wait that ran out."""
import pytest
import torch

gpu = pytest.mark.gpu


def rand(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").bfloat16()


@pytest.fixture
def withheld():
    """withheld(limit): from here on block 0 leaves its first copy unissued, and waits give up after `limit` polls."""
    from gact import _native as nv
    yield lambda limit: nv.lib.gact_pipeline_test_hook(limit, 1)
    nv.lib.gact_pipeline_test_hook(0, 0)
    torch.cuda.synchronize()
    nv.lib.gact_pipeline_error_reset()


@gpu
def test_every_limit_is_taken_as_it_is_given(withheld):
    """A wait's time grows with its polls: 2^20 of them (the quantizer's default) take four times as long as 2^18, not more than twice that."""
    from gact import fused
    x, w = rand(100, 256), rand(64, 256, seed=1)
    fused.op_linear(x, w, save=False)

    def ms(limit):
        from gact import _native as nv
        torch.cuda.synchronize()
        withheld(limit)
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        fused.op_linear(x, w, save=False)
        b.record()
        torch.cuda.synchronize()
        nv.lib.gact_pipeline_error_reset()
        return a.elapsed_time(b)

    short = ms(1 << 18)
    assert 2 * short < ms(1 << 20) < 8 * short
