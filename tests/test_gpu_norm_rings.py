"""Layer norm's backward pass through rings of copies: sizes on both sides of the rule that picks them, every type, rows that are part of
a larger tensor, single gradients; and the rings where only the diagnostics hook puts them."""
import pytest
import torch

from test_gpu_fused import check_norm

gpu = pytest.mark.gpu


def rand(*shape, seed=0, dtype=torch.bfloat16, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").mul_(std).to(dtype)


@gpu
@pytest.mark.parametrize("dtype,rows,cols", [(torch.bfloat16, 4736, 2056), (torch.bfloat16, 4737, 2056), (torch.float16, 5001, 3200), (torch.bfloat16, 6000, 4096),
                                             (torch.float16, 4800, 4104), (torch.float32, 14209, 2056), (torch.bfloat16, 4801, 2048), (torch.bfloat16, 4900, 2060)])
def test_many_long_rows(dtype, rows, cols):
    x = rand(rows, cols, seed=1, dtype=dtype) * 2 + 0.5
    w, b = rand(cols, seed=2, std=0.2, dtype=dtype) + 1, rand(cols, seed=3, std=0.3, dtype=dtype)
    check_norm(x, w, b, rand(rows, cols, seed=4, std=0.1, dtype=dtype), 1e-5, True)


@gpu
def test_many_long_rows_of_a_larger_tensor():
    big, gy = rand(5000, 2600, seed=1), rand(5000, 2600, seed=2, std=0.1)
    w, b = rand(2400, seed=3, dtype=torch.float32) + 1, rand(2400, seed=4, dtype=torch.float32)
    x, dy = big[:, 8:2408], gy[:, 16:2416]
    check_norm(x, w, b, dy, 1e-5, True)
    check_norm(x, None, None, dy, 1e-5, True, (True, False, False))
    check_norm(x, w, None, dy, 1e-5, True, (False, True, False))
    check_norm(x, None, b, dy, 1e-5, True, (False, False, True))


@gpu
@pytest.mark.parametrize("rows,cols", [(1, 8), (3, 64), (700, 264), (2000, 2048), (500, 4096)])
def test_rings_where_only_the_hook_puts_them(rows, cols):
    """The hook withholds block 0's first copy: row 0 and the rows behind it in that block are lost and reported, every other block's rows
    come out right."""
    from gact import _native as nv, fused
    x, w = rand(rows, cols, seed=1), rand(cols, seed=2)
    _, s = fused.op_layer_norm(x, w)
    dy = rand(rows, cols, seed=3)
    want = fused.op_layer_norm_backward(dy, s, (True, False, False))[0]
    nv.lib.gact_pipeline_test_hook(2000, 1)
    try:
        got = fused.op_layer_norm_backward(dy, s)[0]
        torch.cuda.synchronize()
    finally:
        nv.lib.gact_pipeline_test_hook(0, 0)
    with pytest.raises(RuntimeError, match="did not arrive"):
        fused.check()
    blocks = min(rows, 4 * torch.cuda.get_device_properties(0).multi_processor_count)
    fine = torch.arange(rows, device="cuda") % blocks != 0
    # (sums in another order: at most a step of the stored type, 2^-7 of the value, and 64 steps of fp32 of the row's largest)
    a, b = got[fine].double(), want[fine].double()
    assert bool(((a - b).abs() <= 2.0 ** -7 * b.abs() + 64 * 2.0 ** -24 * 100).all())
