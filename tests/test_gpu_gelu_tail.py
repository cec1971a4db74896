"""GELU far below zero, relative to its own tiny values."""
import math

import pytest
import torch

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_the_negative_tail_of_gelu_relative_to_itself(dtype):
    """Abramowitz & Stegun 7.1.26 evaluated in 64 bits at 2000 points per range is off from Phi by at most the factors here (rounded up);
    to that come half a step of the type and 1e-5 for fp32 (the exponent reaches 122 binades, each argument step 2^-24 of it)."""
    from gact import fused
    one = torch.ones(1, 1, dtype=dtype, device="cuda")
    for lo, hi, off in ((-1, -0.01, 4e-7), (-2, -1, 3.1e-6), (-3, -2, 5.2e-5), (-4, -3, 4.7e-4), (-5, -4, 1.6e-3), (-6, -5, 3.6e-3), (-8, -6, 1.1e-2), (-10, -8, 2e-2),
                        (-12.5, -10, 3.8e-2)):
        x = torch.linspace(lo, hi, 2001).to(dtype).cuda().view(-1, 1)
        z = x.double().cpu()
        want = 0.5 * z * torch.erfc(-z / math.sqrt(2))
        normal = want.abs() >= torch.finfo(dtype).tiny          # (fp16 has subnormals only from about -5 on)
        y = fused.op_linear(x, one, None, "gelu")[0].double().cpu()
        tol = (off + torch.finfo(dtype).eps / 2 + 1e-5) * want.abs()
        assert bool(((y - want).abs() <= tol)[normal].all()), (lo, hi)
        # the slope Phi + z phi changes its sign at -0.75 and grows towards it: compared where the tail has taken over
        if hi <= -2:
            s = fused.op_linear(x, one, None, "gelu", compress=False)[1]
            dx = fused.op_linear_backward(torch.ones_like(x), s, (True, False, False))[0].double().cpu()
            phi = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
            cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
            want = cdf + z * phi
            # dz is rounded and then dx: two half steps
            tol = off * cdf + (torch.finfo(dtype).eps * 1.01 + 1e-5) * want.abs() + 1e-5 * (cdf + z.abs() * phi)
            normal = want.abs() >= torch.finfo(dtype).tiny
            assert bool(((dx - want).abs() <= tol)[normal].all()), (lo, hi)
