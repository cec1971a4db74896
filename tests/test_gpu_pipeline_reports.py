"""Bounded waits of the products and of layer norm's rings: the limit that is asked for, and who learns of a wait that ran out."""
import gc

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


CALLS = ["checkpoint", "restore", "norm", "norm backward", "linear", "linear backward", "replay"]


@gpu
@pytest.mark.parametrize("first", ["linear", "norm backward"])
@pytest.mark.parametrize("second", CALLS)
def test_the_next_call_says_that_a_copy_was_lost(withheld, first, second):
    """No Controller, no level: the call after one that lost a copy raises, once, whatever it is; check() does too."""
    from gact import _native as nv, fused
    x, w = rand(2000, 2048), rand(64, 2048, seed=1)
    n, norm = fused.op_layer_norm(x)
    y, lin = fused.op_linear(x, w)
    c = fused.op_checkpoint8(x[:4])
    calls = {"checkpoint": lambda: fused.op_checkpoint8(x[:4]).buf, "restore": lambda: fused.op_restore8(c), "norm": lambda: fused.op_layer_norm(x[:4])[0],
             "norm backward": lambda: fused.op_layer_norm_backward(x, norm)[0], "linear": lambda: fused.op_linear(x, w)[0],
             "linear backward": lambda: fused.op_linear_backward(y, lin)[1]}
    gc.collect()                                   # (no graph of another test may be collected inside the capture)
    graph = torch.cuda.CUDAGraph()
    norm_call = calls["norm"]
    with torch.cuda.graph(graph):
        captured = norm_call()
    calls["replay"] = lambda: (graph.replay(), norm_call(), captured)[2]
    want = {k: f().clone() for k, f in calls.items()}
    torch.cuda.synchronize()
    withheld(2000)
    calls[first]()
    torch.cuda.synchronize()
    nv.lib.gact_pipeline_test_hook(0, 0)
    with pytest.raises(RuntimeError, match="did not arrive"):
        calls[second]()
    assert torch.equal(calls[second](), want[second])
    with pytest.raises(RuntimeError, match="did not arrive"):
        fused.check()
    fused.check()
    assert torch.equal(calls[first](), want[first])


@gpu
def test_check_without_another_call(withheld):
    from gact import _native as nv, fused
    x, w = rand(100, 256), rand(64, 256, seed=1)
    withheld(2000)
    fused.op_linear(x, w, save=False)
    nv.lib.gact_pipeline_test_hook(0, 0)
    with pytest.raises(RuntimeError, match="did not arrive"):
        fused.check()
    fused.op_linear(x, w, save=False)              # (said once)
    fused.check()


@gpu
def test_a_controller_without_compression_reports_too(withheld):
    import gact
    from gact import fused
    gact.set_optimization_level("L0")
    c = gact.Controller(torch.nn.Linear(2, 2))
    c.install_hook()
    x, w = rand(100, 256), rand(64, 256, seed=1)
    withheld(2000)
    fused.op_linear(x, w, save=False)
    with pytest.raises(RuntimeError, match="did not arrive"):
        c.uninstall_hook()
