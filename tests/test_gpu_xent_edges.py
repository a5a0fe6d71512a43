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


@gpu
@pytest.mark.parametrize("V", [200, 700])
def test_operands_near_the_ends_of_the_range(V):
    x, w, t = _case(90, 128, V, torch.float32, 3)
    for size in (1e33, 1e35):
        _check(x * size, w / size, t)
        _check(x / size, w * size, t)
    for size in (1e37, 1e40):  # subnormal on one side: the losses
        small = w.double() / size
        _check(x * 1e37, small.float(), t, need=(False, False))
        _check((x.double() / size).float(), w * 1e37, t, need=(False, False))
    _check(x * 1e-35, w * 1e-35, t, need=(False, False))
    _check(x * 1e-43, w, t, need=(False, False))


@gpu
@pytest.mark.parametrize("V", [200, 700])
def test_gradients_that_need_both_ends(V):
    """The weight is subnormal and the gradient that comes in large, or the other way round: what goes out is in
    the middle of the range.  dx = grad * (softmax - onehot) . w; at a constant x every softmax is 1 / V."""
    import sparsecore_b200 as sl

    g = torch.Generator().manual_seed(4)
    w = (torch.randn(V, 64, generator=g).double() * 1e-38).float().to(dev())
    x = torch.zeros(50, 64, device=dev(), requires_grad=True)
    t = torch.randint(0, V, (50,), generator=g).to(dev())
    for grad, weight in ((1e30, w), (1e-30, w * 1e30 * 1e38)):
        (dx,) = torch.autograd.grad(sl.linear_cross_entropy(x, weight, t, reduction="sum"), (x,), torch.tensor(grad, device=dev()))
        ref = grad * (weight.double().mean(0) - weight.double()[t])
        # 2^-22 an operand, and sums of V
        lim = (16 + V / 8) * 2.0 ** -24 * grad * (weight.double().abs().mean(0) + weight.double()[t].abs()) + 2.0 ** -39 * grad * float(weight.abs().max()) * V
        assert bool(((dx.double() - ref).abs() <= lim).all())


@gpu
def test_columns_whose_logits_are_minus_infinity():
    """A stretch of the vocabulary that cannot be chosen adds nothing to the sum."""
    import sparsecore_b200 as sl

    x, w, t = _case(60, 64, 1000, torch.bfloat16, 5, ignored=0)
    x = x.abs() + 0.01
    w[300:] = -math.inf
    t = t % 300
    got = sl.linear_cross_entropy(x, w, t, reduction="none")
    want = sl.linear_cross_entropy(x, w[:300].contiguous(), t, reduction="none")
    assert bool(((got - want).abs() <= 16 * 2.0 ** -24 * (1 + want.abs())).all())


@gpu
def test_long_sums_of_one_sign_do_not_drift():
    """2^18 tokens with one target: dW is a sum of terms of one sign, and cutting
    at each addition would show as a drift of n / 4 steps of 2^-23 (n sums of 16).
    softmax is 1 / 1024 everywhere, so the target's gradient -1023/1024 is held
    exactly; what is left is the output's rounding, which has no sign: over 4096
    columns its mean is below 2^-12 / 64 * 4."""
    import sparsecore_b200 as sl

    T, D, V = 1 << 18, 4096, 1024
    g = torch.Generator(device=dev()).manual_seed(6)
    x = torch.rand(T, D, generator=g, device=dev(), dtype=torch.float16).add_(0.5).requires_grad_(False)
    w = torch.zeros(V, D, device=dev(), dtype=torch.float16, requires_grad=True)
    t = torch.full((T,), 7, dtype=torch.int64, device=dev())
    (dw,) = torch.autograd.grad(sl.linear_cross_entropy(x, w, t), (w,))
    total = torch.zeros(D, dtype=torch.float64, device=dev())
    for a in range(0, T, 8192):
        total += x[a:a + 8192].double().sum(0)
    ref = -1023 / 1024 * total / T
    drift = float(((dw[7].double() - ref) / ref).mean())
    assert abs(drift) <= 2.0 ** -16, drift


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [70, 600])
@pytest.mark.parametrize("was,now", [(0, 1), (1, 0), (0, 0), (1, 1)])
def test_saved_tensors_that_come_back_elsewhere(dtype, V, was, now):
    """Hooks may put what is kept for the backward pass away and bring it back at another address."""
    import sparsecore_b200 as sl

    def at(v, off):
        n = v.numel()
        return torch.empty(n + 8, dtype=v.dtype, device=dev())[off:off + n].view(v.shape).copy_(v)

    x, w, t = _case(130, 64, V, dtype, 8)
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    want = torch.autograd.grad(sl.linear_cross_entropy(xr, wr, t), (xr, wr))
    xl, wl = at(x, was).requires_grad_(), at(w, was).requires_grad_()

    def back(v):
        return at(v.to(dev()), now) if v.dim() == 2 else v.to(dev())

    with torch.autograd.graph.saved_tensors_hooks(lambda v: v.cpu(), back):
        loss = sl.linear_cross_entropy(xl, wl, t)
    got = torch.autograd.grad(loss, (xl, wl))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_a_call_without_gradients_keeps_no_room_for_them():
    """Of a vocabulary of one tile only a training call keeps the logits' gradient."""
    from sparsecore_b200 import loss as L

    x, w = torch.zeros(20000, 64, device=dev()), torch.zeros(200, 64, device=dev())
    kept = {train: L._sizes(x, w, 0, train)[0] for train in (0, 1)}
    assert kept[1] - kept[0] >= 20000 * 200 * 2 * 2


@gpu
def test_forward_mode_is_refused():
    """Tangents have no way through; a result without one would be wrong in silence."""
    import torch.autograd.forward_ad as fw

    import sparsecore_b200 as sl

    x, w, t = _case(8, 16, 20, torch.float32, 9)
    n = torch.ones(16, device=dev())
    with fw.dual_level():
        d, dw, dn = (fw.make_dual(v, torch.ones_like(v)) for v in (x, w, n))
        for call in (lambda: sl.linear_cross_entropy(d, w, t), lambda: sl.linear_cross_entropy(x, dw, t),
                     lambda: sl.residual_norm(d, x, n), lambda: sl.residual_norm(x, x, n, gate=dn),
                     lambda: sl.residual_norm(x, x, n, scale=fw.make_dual(torch.ones(1, device=dev()), torch.ones(1, device=dev())))):
            with pytest.raises(RuntimeError, match="forward"):
                call()
        sl.linear_cross_entropy(x, w, t)  # what has no tangent goes through
        sl.residual_norm(x, x, n)
