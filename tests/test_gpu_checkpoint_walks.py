"""Checkpoints of rows that do not start on 16-byte boundaries, at row lengths on both sides of every choice of walk."""
import pytest
import torch

from test_gpu_fused import kept64, same

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("cols", [1, 31, 33, 71, 72, 73, 127, 129, 161, 191, 193, 255, 257, 383, 385, 511, 513, 575, 577, 769, 1025])
def test_odd_rows_are_exact(cols, dtype):
    from gact import fused
    g = torch.Generator(device="cuda").manual_seed(cols)
    for rows in (3, 1 + 20000 // cols):
        x = torch.randn(rows, cols + 1, generator=g, device="cuda").to(dtype)
        x.view(-1)[::7] *= 30.0
        for v in (x[:, :cols], x[:, 1:], x[:, :cols].contiguous()):
            c = fused.op_checkpoint8(v)
            assert same(fused.op_restore8(c), kept64(v)) and same(fused.op_restore8(c, torch.float32), kept64(v))
            assert not c.codes[:, cols:].any()


@gpu
@pytest.mark.parametrize("cols", [71, 129, 191, 193, 257])
def test_large_tensors_of_odd_rows_are_exact(cols):
    """Enough rows for four chunks a thread."""
    from gact import fused
    g = torch.Generator(device="cuda").manual_seed(cols)
    rows = 12000000 // cols
    x = torch.randn(rows, cols, generator=g, device="cuda").bfloat16()
    c = fused.op_checkpoint8(x)
    y = fused.op_restore8(c)
    for lo in (0, rows // 2, rows - 700):
        assert same(y[lo:lo + 700], kept64(x[lo:lo + 700]))
    small = fused.op_checkpoint8(x[-1000:])
    assert torch.equal(c.codes[-1000:], small.codes) and torch.equal(c.scales[-1000:], small.scales)
    # (padded rows on 16-byte boundaries take the other kernels; the last block is padded with zeros either way)
    padded = torch.nn.functional.pad(x, (0, (-cols) % 32))
    assert torch.equal(fused.op_checkpoint8(padded).buf, c.buf)
