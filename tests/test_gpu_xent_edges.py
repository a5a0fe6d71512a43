"""linear_cross_entropy at the ends of its operands' and gradients' ranges.
Tolerances as in test_gpu_xent where no other is derived."""
import math

import pytest
import torch

from gpu_helpers import dev
from test_gpu_xent import _case, _check

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [90, 700])
def test_gradients_of_single_losses_that_are_not_finite(dtype, V):
    """What is not finite on its way in is not finite on its way out: a step with
    an overflowed loss scale must be seen as one."""
    import sparsecore_b200 as sl

    x, w, t = _case(40, 64, V, dtype, 1, ignored=0)
    t[3] = -100
    for fill, rest in ((math.inf, math.inf), (math.nan, math.nan), (math.inf, 0.0), (math.nan, 0.0), (-math.inf, 1.0)):
        xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
        grad = torch.full((40,), rest, device=dev())
        grad[:20] = fill
        dx, dw = torch.autograd.grad(sl.linear_cross_entropy(xl, wl, t, reduction="none"), (xl, wl), grad)
        bad = ~torch.isfinite(grad)
        bad[3] = False  # its loss counts for nothing, whatever comes in
        assert torch.equal((~torch.isfinite(dx)).any(1), bad)
        assert not dx[3].any()
        if rest == 0.0:
            assert not dx[20:].any()
        assert not torch.isfinite(dw).any()


@gpu
@pytest.mark.parametrize("V", [200, 300, 384])
def test_operands_that_are_both_tiny(V):
    x, w, t = _case(90, 128, V, torch.float32, 2)
    _check(x * 1e-20, w * 1e-20, t)
    _check(x * 1e-30, w * 1e-5, t)
