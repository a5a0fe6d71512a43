"""linear_cross_entropy against its formula in 64 bits: losses and both gradients
over types, odd sizes, reductions, ignored and bad targets, and graph replay.

Tolerances by arithmetic.  A logit is a sum of D products; an operand held as two
fp16 planes is off by 2^-22 of it, and every 16 products are added to the sum
with at most one step of 2^-23: dz = (64 + D / 8) * 2^-24 * sum |x| |w| bounds it.
A probability is off by 4 dz of it and a few steps of the exponential; the
logits' gradient is then held in bf16, fp16, or two planes of fp16 (half a
step: 2^-8, 2^-11, 2^-22 of it, and 2^-39 of absolute spacing in fp16).  These
roundings are independent of each other, so a sum of n of them is held to eight
times the root of the sum of their squares; errors of one sign are added up in
full; and rounding to the output's type adds half a step."""
import pytest
import torch

from gpu_helpers import dev

gpu = pytest.mark.gpu
U = 2.0 ** -24
HELD = {torch.float32: 2.0 ** -22, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _case(T, D, V, dtype, seed, ignored=0.1, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, D, generator=g).to(dtype).to(dev())
    w = (torch.randn(V, D, generator=g) * (scale / D ** 0.5)).to(dtype).to(dev())
    t = torch.randint(0, V, (T,), generator=g)
    t[torch.rand(T, generator=g) < ignored] = -100
    return x, w, t.to(dev())


def _check(x, w, t, reduction="mean", ignore=-100, grad=None, need=(True, True)):
    import sparsecore_b200 as sl

    xl, wl = x.clone().requires_grad_(need[0]), w.clone().requires_grad_(need[1])
    loss = sl.linear_cross_entropy(xl, wl, t, ignore_index=ignore, reduction=reduction)
    assert loss.dtype == torch.float32
    D, V, keep = x.shape[-1], w.shape[0], t != ignore
    xd, wd = torch.where(keep[:, None], x.double(), 0.0), w.double()
    z = xd @ wd.t()
    dz = ((64 + D / 8) * U * (xd.abs() @ wd.abs().t())).amax(1)
    lse = torch.logsumexp(z, 1)
    at = t.clamp_min(0)
    each = torch.where(keep, lse - z.gather(1, at[:, None])[:, 0], 0.0)
    lim = torch.where(keep, 2 * dz + 16 * U * (1 + lse.abs() + each.abs()), 0.0)
    n = keep.sum()
    if reduction == "none":
        assert bool(((loss.double() - each).abs() <= lim).all())
    elif reduction == "mean" and int(n) == 0:
        assert torch.isnan(loss)  # the mean of nothing; its gradients are zero
    else:
        over = n if reduction == "mean" else 1
        assert abs(float(loss.double() - each.sum() / over)) <= float((lim.sum() + U * each.sum()) / over)
    if not any(need):
        return loss
    if grad is None:
        grad = torch.ones_like(loss)
    got = torch.autograd.grad(loss, [v for v, k in zip((xl, wl), need) if k], grad)
    got = dict(zip([k for k, on in zip("xw", need) if on], got))
    p = torch.exp(z - lse[:, None])
    gt = grad.double().expand(t.shape) * (keep / n.clamp_min(1) if reduction == "mean" else keep)
    G = p.clone()
    G[torch.arange(len(t), device=t.device), at] -= 1
    G = G * gt[:, None]
    top = float(gt.abs().max())
    held = HELD[x.dtype] * G.abs() + 2.0 ** -39 * top
    shift = p * (4 * dz[:, None] + 32 * U) * gt.abs()[:, None]  # the row's error of one sign
    half = torch.finfo(x.dtype).eps / 2
    # fp16 outputs below the smallest normal are spaced evenly
    floor = 2.0 ** -24 if x.dtype == torch.float16 else 0.0
    for key, a, b, h, s in (("x", G, wd, held, shift), ("w", G.t(), xd, held.t(), shift.t())):
        if key not in got:
            continue
        ref = a @ b
        k = a.shape[1]
        lim = 8 * torch.sqrt((h ** 2) @ (b ** 2)) + s @ b.abs() + (64 + k / 8) * U * (a.abs() @ b.abs())
        lim = lim + half * (ref.abs() + lim) + floor
        d = (got[key].double() - ref).abs()
        assert got[key].dtype == x.dtype and got[key].shape == ref.shape
        assert bool((d <= lim).all()), f"d{key} off by {float((d / lim.clamp_min(1e-300)).max()):.3g} times the bound"
    return loss


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,D,V", [(1, 1, 1), (1, 64, 2), (3, 7, 5), (2, 768, 256), (129, 65, 65), (255, 64, 257), (256, 128, 256),
                                   (257, 200, 513), (700, 384, 65), (64, 1000, 3001), (33, 1024, 4099), (1500, 96, 1031)])
def test_sizes_and_types(T, D, V, dtype):
    _check(*_case(T, D, V, dtype, T + D + V))


@gpu
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_reductions(reduction, dtype):
    x, w, t = _case(150, 96, 300, dtype, 1)
    g = torch.Generator().manual_seed(2)
    grad = torch.randn((150,) if reduction == "none" else (), generator=g).to(dev())
    if reduction == "none":
        grad[5] = 0.0
        grad[7] = 1e-3
    _check(x, w, t, reduction, grad=grad)
    _check(x, w, t, reduction, grad=torch.zeros_like(grad))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_gradient_or_none(dtype):
    c = _case(70, 128, 500, dtype, 3)
    for need in ((True, False), (False, True), (False, False)):
        _check(*c, need=need)


@gpu
def test_pieces_of_the_vocabulary():
    """Enough tokens for the gradient to be taken in one large piece, and in several (planes above 512 MB)."""
    _check(*_case(17000, 40, 8300, torch.float32, 18))
    _check(*_case(40000, 33, 7001, torch.bfloat16, 19))
    _check(*_case(17000, 256, 8300, torch.float32, 20))
    _check(*_case(9000, 64, 8300, torch.float32, 4))
    _check(*_case(20000, 40, 7000, torch.bfloat16, 5))


@gpu
def test_long_sums_of_few_columns():
    """A small vocabulary under many tokens: the weight's gradient is one long sum a column."""
    _check(*_case(16384, 384, 65, torch.float32, 6))
    _check(*_case(16001, 104, 3, torch.float16, 7))


@gpu
@pytest.mark.parametrize("scale", [1e-3, 30.0, 300.0])
def test_flat_and_sharp_logits(scale):
    for dtype in (torch.float32, torch.bfloat16):
        _check(*_case(130, 256, 700, dtype, 8, scale=scale))


@gpu
@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e6, 1e15])
def test_operands_of_any_size(size):
    """32-bit operands are scaled into fp16's range: tiny and huge ones keep their digits."""
    x, w, t = _case(90, 128, 200, torch.float32, 9)
    _check(x * size, w / size, t)
    _check(x / size, w * size, t)


@gpu
def test_rows_of_very_different_size():
    x, w, t = _case(90, 128, 200, torch.float32, 10)
    x[::3] *= 1e-3
    w[::5] *= 1e-4
    w[7] = 0
    x[6] = 0
    _check(x, w, t)


@gpu
def test_ignored_tokens_count_for_nothing():
    import sparsecore_b200 as sl

    for dtype in (torch.float32, torch.bfloat16):
        x, w, t = _case(40, 64, 100, dtype, 11, ignored=0.5)
        x[t == -100] = float("nan")
        x[t == -100] = float("inf")
        _check(x, w, t)
        t = torch.where(t == -100, 3, t)
        _check(x.nan_to_num(0, 0, 0), w, t, ignore=3)
        xl, wl = x.nan_to_num(0, 0, 0).requires_grad_(), w.clone().requires_grad_()
        loss = sl.linear_cross_entropy(xl, wl, torch.full_like(t, -100))
        assert torch.isnan(loss)
        loss.backward()
        assert not xl.grad.any() and not wl.grad.any()
        assert sl.linear_cross_entropy(xl, wl, torch.full_like(t, -100), reduction="sum") == 0


@gpu
def test_targets_outside_the_vocabulary():
    import sparsecore_b200 as sl

    x, w, t = _case(40, 64, 100, torch.float32, 12)
    t[3], t[9], t[11] = 100, -1, 1 << 40
    xl = x.clone().requires_grad_()
    loss = sl.linear_cross_entropy(xl, w, t, reduction="none")
    bad = torch.zeros(40, dtype=torch.bool, device=dev())
    bad[[3, 9, 11]] = True
    assert torch.equal(torch.isnan(loss), bad)
    loss.sum().backward()
    assert torch.equal(torch.isnan(xl.grad).all(1), bad) and torch.isfinite(xl.grad[~bad]).all()
    assert torch.isnan(sl.linear_cross_entropy(x, w, t))


@gpu
def test_values_that_are_not_finite_reach_their_row():
    import sparsecore_b200 as sl

    x, w, t = _case(40, 64, 100, torch.float32, 13, ignored=0)
    clean = sl.linear_cross_entropy(x, w, t, reduction="none")
    x[5, 2] = float("nan")
    x[8, 0] = float("inf")
    loss = sl.linear_cross_entropy(x, w, t, reduction="none")
    assert torch.isnan(loss[[5, 8]]).all()
    rest = [i for i in range(40) if i not in (5, 8)]
    assert torch.equal(loss[rest], clean[rest])


@gpu
def test_gradients_against_differences():
    """The formula in 64 bits, differenced at +-1e-6 along one direction in x and w at once."""
    import sparsecore_b200 as sl

    x, w, t = _case(60, 80, 150, torch.float32, 14)
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    gx, gw = torch.autograd.grad(sl.linear_cross_entropy(xl, wl, t), (xl, wl))
    g = torch.Generator(device=dev()).manual_seed(1)
    a, b = (torch.randn(v.shape, generator=g, device=dev()).double() for v in (x, w))

    def f(e):
        z = (x.double() + e * a) @ (w.double() + e * b).t()
        keep = t != -100
        return (torch.logsumexp(z, 1) - z.gather(1, t.clamp_min(0)[:, None])[:, 0])[keep].mean()

    slope = float((f(1e-6) - f(-1e-6)) / 2e-6)
    terms = torch.cat([(gx.double() * a).view(-1), (gw.double() * b).view(-1)])
    assert abs(float(terms.sum()) - slope) <= float(terms.abs().sum()) * 256 * U + 1e-8


@gpu
def test_strides_and_leading_dimensions():
    import sparsecore_b200 as sl

    x, w, t = _case(60, 72, 90, torch.bfloat16, 15)
    want = sl.linear_cross_entropy(x, w, t, reduction="none")
    wide = torch.zeros(60, 73, dtype=torch.bfloat16, device=dev())
    wide[:, 1:] = x
    off = torch.empty(90 * 72 + 1, dtype=torch.bfloat16, device=dev())[1:].view(90, 72)
    off.copy_(w)
    t2 = torch.stack([t, t], 1)[:, 0]
    assert torch.equal(sl.linear_cross_entropy(wide[:, 1:], off, t2, reduction="none"), want)
    assert torch.equal(sl.linear_cross_entropy(x.t().contiguous().t(), w.t().contiguous().t(), t, reduction="none"), want)
    cube = sl.linear_cross_entropy(x.view(3, 20, 72), w, t.view(3, 20), reduction="none")
    assert cube.shape == (3, 20) and torch.equal(cube.view(-1), want)
    one = sl.linear_cross_entropy(x[1], w, t[1], reduction="none")
    assert one.shape == () and torch.equal(one, want[1])


@gpu
def test_no_tokens():
    import sparsecore_b200 as sl

    x, w = torch.zeros(0, 16, device=dev(), requires_grad=True), torch.zeros(9, 16, device=dev(), requires_grad=True)
    t = torch.zeros(0, dtype=torch.int64, device=dev())
    assert torch.isnan(sl.linear_cross_entropy(x, w, t)) and sl.linear_cross_entropy(x, w, t, reduction="none").shape == (0,)
    sl.linear_cross_entropy(x, w, t, reduction="sum").backward()
    assert x.grad.shape == (0, 16) and not w.grad.any()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_runs_are_repeatable_side_by_side_and_replay(dtype):
    import sparsecore_b200 as sl

    x, w, t = _case(300, 128, 1000, dtype, 16)
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()

    def once():
        loss = sl.linear_cross_entropy(xl, wl, t)
        return [loss.detach(), *torch.autograd.grad(loss, (xl, wl))]

    first, second = once(), once()
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    # two at once, on two streams
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        third = once()
    fourth = once()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(first, third, fourth))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once()
    with torch.no_grad():
        xl.mul_(0.5)
        t[0] = -100
    want = once()
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, want))


@gpu
def test_the_backward_pass_can_be_taken_twice():
    import sparsecore_b200 as sl

    x, w, t = _case(50, 64, 80, torch.float32, 17)
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = sl.linear_cross_entropy(xl, wl, t)
    a = torch.autograd.grad(loss, (xl, wl), retain_graph=True)
    b = torch.autograd.grad(loss, (xl, wl), torch.tensor(2.0, device=dev()))
    assert torch.equal(2 * a[0], b[0]) and torch.equal(2 * a[1], b[1])


def test_refusals_without_a_gpu():
    import sparsecore_b200 as sl

    x, w, t = torch.zeros(3, 4), torch.zeros(5, 4), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        sl.linear_cross_entropy(x, w, t)
    with pytest.raises(TypeError):
        sl.linear_cross_entropy(x, w, [0, 0, 0])
    with pytest.raises(ValueError, match="reduction"):
        sl.linear_cross_entropy(x, w, t, reduction="max")


@gpu
def test_refusals():
    import sparsecore_b200 as sl

    x, w, t = (v.to(dev()) for v in (torch.zeros(3, 4), torch.zeros(5, 4), torch.zeros(3, dtype=torch.int64)))
    for bad in ((x.double(), w.double(), t), (x, w.half(), t), (x, w[:, :3], t), (x, w, t[:2]), (x, w, t.int()), (x, w[:0], t),
                (x, w.view(-1), t)):
        with pytest.raises(ValueError):
            sl.linear_cross_entropy(*bad)
    with pytest.raises(RuntimeError):
        sl.linear_cross_entropy(x, w.cpu(), t)


@gpu
@pytest.mark.parametrize("vocab", [70, 600])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_between_other_work(dtype, vocab):
    """The kernels of a pass may start before the one ahead of them ends: what
    lies before and behind them (a fill, a copy, another stream's work, the
    reuse of their buffers) is ordered all the same, eager and captured."""
    import sparsecore_b200 as sl

    x, w, t = _case(300, 136, vocab, dtype, 23)
    xl, wl = torch.zeros_like(x).requires_grad_(), torch.zeros_like(w).requires_grad_()
    tl = torch.zeros_like(t)
    side = torch.cuda.Stream()

    def once():
        with torch.no_grad():
            wl.zero_()  # a fill, a copy and a kernel of another stream write the operands
            xl.copy_(x)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                wl.add_(w)
                tl.copy_(t)
            torch.cuda.current_stream().wait_stream(side)
        loss = sl.linear_cross_entropy(xl, wl, tl)
        grads = torch.autograd.grad(loss, (xl, wl))
        with torch.no_grad():
            xl.fill_(float("nan"))
            wl.zero_()
            tl.zero_()
            return [loss.detach().clone(), *(g.clone() for g in grads)]

    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = sl.linear_cross_entropy(xr, wr, t)
    want = [loss.detach(), *torch.autograd.grad(loss, (xr, wr))]
    torch.cuda.synchronize()
    for _ in range(20):
        got = once()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once()
    for _ in range(20):
        for h in held:
            h.zero_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
