"""FusedAdamW's step counts, states and rare values: each parameter's own count,
pauses and late starts against torch's AdamW, captured steps, copies and
checkpoints, 8-bit moments at the ends of the range."""
import copy
import math
import pickle

import pytest
import torch

from gpu_helpers import dev

gpu = pytest.mark.gpu


def _params(seed=1, sizes=(70, 300, 5)):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(n, generator=g).to(dev()).requires_grad_() for n in sizes]


def _grads(params, step, on, seed=2):
    g = torch.Generator().manual_seed(seed * 1000 + step)
    for k, p in enumerate(params):
        gr = torch.randn(p.shape, generator=g).to(dev())
        p.grad = gr if k in on else None


# which parameters have a gradient at each step: a late start, pauses, all at once
PATTERNS = [[{0}] * 5 + [{0, 1, 2}] * 4,
            [{0, 1, 2}, {0, 1, 2}, {1, 2}, {0, 1, 2}, {1}, {0, 2}, {0, 1, 2}],
            [set(), {2}, {1}, {0}, {0, 1, 2}, {0, 1}, {0, 1, 2}],
            [{0, 1, 2}, {0}, {0}, {0, 1, 2}, {1, 2}, {0, 1, 2}]]


@gpu
@pytest.mark.parametrize("pattern", PATTERNS)
@pytest.mark.parametrize("capturable", [False, True])
def test_each_parameter_counts_its_own_steps(pattern, capturable):
    import sparsecore_b200 as sl

    a, b = _params(), _params()
    kw = dict(lr=1e-2, betas=(0.9, 0.99), weight_decay=0.05)
    oa, ob = torch.optim.AdamW(a, **kw), sl.FusedAdamW(b, capturable=capturable, **kw)
    for step, on in enumerate(pattern):
        _grads(a, step, on)
        _grads(b, step, on)
        oa.step()
        ob.step()
        for p, q in zip(a, b):
            torch.testing.assert_close(q, p, rtol=1e-5, atol=1e-6)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_the_first_step_of_a_late_parameter_is_the_learning_rate(bits):
    """m / root of a first step is 1 whatever the gradient is, to the rounding of
    32-bit numbers (the 8-bit step takes its quotient to 2^-22)."""
    import sparsecore_b200 as sl

    params = _params()
    opt = sl.FusedAdamW(params, lr=1e-2, weight_decay=0.0, state_bits=bits)
    for step in range(300):
        _grads(params, step, {0, 2})
        opt.step()
    before = params[1].detach().clone()
    _grads(params, 300, {0, 1, 2})
    opt.step()
    moved = (params[1].detach() - before).abs().double()
    big = params[1].grad.abs() > 1e-3  # eps is then below 1e-5 of the root
    assert bool(((moved[big] - 1e-2).abs() <= 1e-2 * 2e-5 + 2.0 ** -23 * before[big].abs()).all())


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
def test_a_layer_drawn_again_starts_its_count_again(bits, capturable):
    import sparsecore_b200 as sl

    torch.manual_seed(3)
    model = torch.nn.Sequential(sl.SparseLinear(96, 64, sparsity=0.8, device=dev()), torch.nn.Linear(64, 8).to(dev()))
    # after 50 steps the old count's corrections make a first step 0.5 / sqrt(0.001 / (1 - 0.999^51)) = 3.5 times lr
    opt = sl.FusedAdamW(model, lr=1e-3, betas=(0.5, 0.999), weight_decay=0.0, state_bits=bits, capturable=capturable)
    x = torch.randn(40, 96, device=dev())

    def once():
        opt.zero_grad()
        model(x).square().mean().backward()
        opt.step()

    for _ in range(50):
        once()
    n = model[0]._values.numel()
    while model[0]._values.numel() == n:  # until the number of slots is another one
        model[0].reset_parameters()
    before = model[0]._values.detach().clone()
    once()
    assert float((model[0]._values.detach() - before).abs().max()) <= 1e-3 * 1.0001 + 2.0 ** -23
    once()
    assert torch.isfinite(model[0]._values).all()


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_with_a_late_parameter_equal_eager_ones(bits):
    import sparsecore_b200 as sl

    sets = [_params() for _ in range(2)]
    opts = [sl.FusedAdamW(p, lr=1e-2, capturable=True, state_bits=bits) for p in sets]
    fixed = _params(9)
    for p in sets:
        for q, f, k in zip(p, fixed, range(3)):
            q.grad = f.detach().clone() if k != 1 else None
    for _ in range(6):
        for o in opts:
            o.step()
    for p in sets:
        p[1].grad = fixed[1].detach().clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for o in opts:
            o.step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opts[0].step()
    for _ in range(3):
        graph.replay()
        opts[1].step()
    torch.cuda.synchronize()
    for p, q in zip(*sets):
        assert torch.equal(p, q)
    assert int(opts[0].param_groups[0]["step"]) == 10


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
def test_a_state_that_was_on_the_host_goes_on_as_before(bits, capturable, tmp_path):
    """Through a file and back to the host, as checkpoints go, with parameters at different counts."""
    import sparsecore_b200 as sl

    kw = dict(state_bits=bits, capturable=capturable)
    lr = lambda: torch.tensor(1e-2, device=dev()) if capturable else 1e-2  # noqa: E731
    a, b = _params(), _params()
    oa, ob = sl.FusedAdamW(a, lr=lr(), **kw), sl.FusedAdamW(b, lr=lr(), **kw)
    for step, on in enumerate(PATTERNS[1]):
        _grads(a, step, on)
        oa.step()
    torch.save(oa.state_dict(), tmp_path / "opt.pt")
    ob.load_state_dict(torch.load(tmp_path / "opt.pt", map_location="cpu"))
    for group in ob.param_groups:
        for v in (group["step"], group["lr"]):
            assert isinstance(v, torch.Tensor) == capturable and (not capturable or v.device == dev())
    with torch.no_grad():
        for p, q in zip(a, b):
            q.copy_(p)
    for step, on in enumerate(PATTERNS[0], 50):
        for params, o in ((a, oa), (b, ob)):
            _grads(params, step, on)
            o.step()
        for p, q in zip(a, b):
            assert torch.equal(p, q)


@gpu
@pytest.mark.parametrize("capturable", [False, True])
def test_a_state_of_torchs_optimizer_goes_on(capturable):
    import sparsecore_b200 as sl

    a, b = _params(), _params()
    kw = dict(lr=1e-2, betas=(0.9, 0.99), weight_decay=0.05)
    oa = torch.optim.AdamW(a, **kw)
    for step, on in enumerate(PATTERNS[1]):
        _grads(a, step, on)
        oa.step()
    ob = sl.FusedAdamW(b, capturable=capturable, **kw)
    ob.load_state_dict(oa.state_dict())
    with torch.no_grad():
        for p, q in zip(a, b):
            q.copy_(p)
    for step, on in enumerate(PATTERNS[1], 50):
        for params, o in ((a, oa), (b, ob)):
            _grads(params, step, on)
            o.step()
        for p, q in zip(a, b):
            torch.testing.assert_close(q, p, rtol=1e-5, atol=1e-6)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("way", ["copy", "pickle"])
def test_copies_of_an_optimizer_go_on_by_themselves(bits, capturable, way, tmp_path):
    """(torch's 8-bit floats go through its files but not through plain pickle.)"""
    import sparsecore_b200 as sl

    a = _params()
    oa = sl.FusedAdamW(a, lr=1e-2, state_bits=bits, capturable=capturable, seed=3)
    for step, on in enumerate(PATTERNS[1]):
        _grads(a, step, on)
        oa.step()
    if way == "copy":
        ob = copy.deepcopy(oa)
    elif bits == 32:
        ob = pickle.loads(pickle.dumps(oa))
    else:
        torch.save(oa, tmp_path / "opt.pt")
        ob = torch.load(tmp_path / "opt.pt", weights_only=False)
    b = ob.param_groups[0]["params"]
    assert all(p is not q and p.data_ptr() != q.data_ptr() for p, q in zip(a, b))
    for step, on in enumerate(PATTERNS[1], 50):
        for params, o in ((a, oa), (b, ob)):
            _grads(params, step, on)
            o.step()
        for p, q in zip(a, b):
            assert torch.equal(p, q)


@gpu
def test_what_a_capture_would_freeze_is_refused():
    """A count on the host, and moments or counts that begin inside the capture (every replay would begin them again)."""
    import sparsecore_b200 as sl

    params = _params()
    _grads(params, 0, {0, 1, 2})
    opt = sl.FusedAdamW(params, lr=1e-2)
    opt.step()
    keep = [p.detach().clone() for p in params]
    late = _params(5)
    _grads(late, 0, {0, 2})
    opt2 = sl.FusedAdamW(late, lr=1e-2, capturable=True)
    for o, on in ((opt, None), (opt2, None)):
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="captur"):
            with torch.cuda.graph(graph):
                torch.zeros(8, device=dev())
                o.step()
    opt2.step()
    _grads(late, 1, {0, 1, 2})  # a parameter that begins inside the capture
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captur"):
        with torch.cuda.graph(graph):
            torch.zeros(8, device=dev())
            opt2.step()
    _grads(late, 1, {0})  # one that pauses inside it
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captur"):
        with torch.cuda.graph(graph):
            torch.zeros(8, device=dev())
            opt2.step()
    torch.cuda.synchronize()
    assert all(torch.equal(p, k) for p, k in zip(params, keep))


@gpu
def test_a_plan_sees_tensors_that_changed_under_it():
    """Its parameter is cut short where it lies, or replaced; an address in its table is nobody else's."""
    import sparsecore_b200 as sl

    base, m, v = (torch.zeros(64, device=dev()) for _ in range(3))
    p = base.view(64)
    plan = sl.AdamWPlan([p], [m], [v])
    plan.step([torch.ones(64, device=dev())], step=1)
    after = base.clone()
    p.data = p.data[:10]
    with pytest.raises(ValueError, match="elements"):  # its moments are still 64 long
        plan.step([torch.ones(10, device=dev())], step=2)
    m.data, v.data = m.data[:10], v.data[:10]
    plan.step([torch.ones(10, device=dev())], step=2)
    assert not (base[:10] == after[:10]).any() and torch.equal(base[10:], after[10:])
    p, m, v = (torch.zeros(100000, device=dev()) for _ in range(3))
    plan = sl.AdamWPlan([p], [m], [v])
    plan.step([torch.ones(100000, device=dev())], step=1)
    at = p.data_ptr()
    p.data = torch.zeros(10, device=dev())
    m.data, v.data = torch.zeros(10, device=dev()), torch.zeros(10, device=dev())
    others = [torch.zeros(100000, device=dev()) for _ in range(3)]
    assert all(t.data_ptr() != at for t in others)
    plan.step([torch.ones(10, device=dev())], step=1)
    assert p.all() and not any(t.any() for t in others)


@gpu
def test_numbers_made_on_the_device_are_checked():
    import sparsecore_b200 as sl

    p, m, v, g = (torch.zeros(8, device=dev()) for _ in range(4))
    plan = sl.AdamWPlan([p], [m], [v])
    for bad in (torch.zeros(64, dtype=torch.uint8), torch.zeros(4, dtype=torch.uint8, device=dev()), 7,
                torch.zeros(64, dtype=torch.uint8, device=dev())[::2], torch.zeros(65, dtype=torch.uint8, device=dev())[1:]):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            plan.step([g], hyper=bad)
    opt = sl.FusedAdamW([p.requires_grad_()], capturable=True)
    p.grad = g
    opt.step()
    for bad in (torch.zeros((), dtype=torch.int64), torch.zeros((), device=dev()), torch.zeros(2, dtype=torch.int64, device=dev())):
        opt.param_groups[0]["step"] = bad
        with pytest.raises(ValueError):
            opt.step()


def _state8(n):
    z = lambda: torch.zeros(n, dtype=torch.uint8, device=dev()).view(torch.float8_e4m3fn)  # noqa: E731
    return z(), z(), (torch.zeros(-(-n // 256), device=dev()), torch.zeros(-(-n // 256), device=dev()))


@gpu
@pytest.mark.parametrize("n", [256, 300, 2048])
def test_a_second_moment_beyond_32_bits(n):
    """A finite gradient whose square is not: m / sqrt(v) is 0 then and stays it, as with 32-bit moments."""
    import sparsecore_b200 as sl

    kw = dict(lr=1e-3, betas=(0.9, 0.99), weight_decay=0.1)
    g = torch.Generator().manual_seed(n)
    p0 = torch.randn(n, generator=g).to(dev())
    gr = torch.randn(n, generator=g).to(dev())
    p8, p32 = p0.clone(), p0.clone()
    m8, v8, s = _state8(n)
    m32, v32 = torch.zeros(n, device=dev()), torch.zeros(n, device=dev())
    big = torch.zeros(n, dtype=torch.bool, device=dev())
    big[7] = big[n - 1] = True
    for step in (1, 2, 3, 4):
        now = torch.where(big, 3e19 if step == 1 else 0.5, gr)
        sl.adamw_step([p8], [now], [m8], [v8], step=step, scales=[s], **kw)
        sl.adamw_step([p32], [now], [m32], [v32], step=step, **kw)
        assert torch.isfinite(p8).all() and torch.isfinite(s[0]).all() and torch.isfinite(s[1]).all()
        assert torch.equal(p8[big], p32[big])
        assert torch.isinf(v32[big]).all()
    opt = sl.FusedAdamW([p8.requires_grad_()], state_bits=8)
    opt.state[p8].update(exp_avg=m8, exp_avg_sq_root=v8, exp_avg_scale=s[0], exp_avg_sq_root_scale=s[1])
    m, v = opt.state_values(p8)
    assert torch.equal(torch.isinf(v), big) and torch.isfinite(m).all()


@gpu
@pytest.mark.parametrize("n", [512, 4096])
@pytest.mark.parametrize("eps", [0.0, 1e-8])
def test_second_moments_below_the_normal_range(n, eps):
    """Gradients of 1e-20: v is subnormal, its root is not.  One step from nothing, in 32-bit operations: 16 roundings
    (the root of a subnormal v is taken of the rounded v)."""
    import sparsecore_b200 as sl

    g = torch.Generator().manual_seed(8)
    gr = (torch.rand(n, generator=g).double() * 4e-20 + 1e-21).float().to(dev())
    gr[256:300] = 0.3  # a block with ordinary ones beside them
    p = torch.zeros(n, device=dev())
    m, v, s = _state8(n)
    sl.adamw_step([p], [gr], [m], [v], step=1, scales=[s], lr=1.0, betas=(0.9, 0.99), eps=eps, weight_decay=0.0)
    root = (gr * gr * torch.tensor(1 - 0.99, device=dev())).sqrt()
    m1 = gr * torch.tensor(1 - 0.9, device=dev())
    want = -(m1.double() / (1 - 0.9)) / (root.double() / math.sqrt(1 - 0.99) + eps)
    assert bool(((p.double() - want).abs() <= 16 * 2.0 ** -24 * want.abs()).all())
    top = root.view(-1, 256).amax(1).clamp_min(2.0 ** -100)
    torch.testing.assert_close(s[1], top / 448, rtol=1e-6, atol=0)
    held, step = v.float() * s[1].repeat_interleave(256), s[1].repeat_interleave(256) * 2.0 ** -9
    assert bool(((held - root).abs() <= root / 8 * 1.001 + step).all()) and bool((held > 0).all())


@gpu
def test_groups_that_take_turns_keep_their_tables():
    """And a step that is refused counts for nothing."""
    import sparsecore_b200 as sl

    for capturable in (False, True):
        a, b = _params(1), _params(2)
        opt = sl.FusedAdamW([{"params": a}, {"params": b}], lr=1e-2, capturable=capturable)
        seen = []
        for step in range(6):
            now, rest = (a, b) if step % 2 == 0 else (b, a)
            _grads(now, step, {0, 1, 2})
            _grads(rest, step, set())
            opt.step()
            seen.append(dict(opt._plans))
        assert seen[1] == seen[5]
        _grads(a, 7, {0, 1, 2})
        _grads(b, 7, set())
        a[1].grad = None
        a[1].data = a[1].data[:5]  # its moments are longer
        count, keep = int(opt.param_groups[0]["step"]), a[0].detach().clone()
        a[1].grad = torch.ones(5, device=dev())
        opt.state[a[1]]["exp_avg"].data = torch.zeros(5, device=dev())
        with pytest.raises(ValueError):
            opt.step()
        assert int(opt.param_groups[0]["step"]) == count and torch.equal(a[0], keep)


@gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("n", [300, 2048])
def test_neighbours_of_what_is_not_finite_are_what_they_would_be(n, bad):
    """Bit for bit: the largest of the block, which its scale is of, is another element."""
    import sparsecore_b200 as sl

    g = torch.Generator().manual_seed(12)
    p0, gr = torch.randn(n, generator=g).to(dev()), torch.randn(n, generator=g).to(dev())
    gr[9] = 20.0
    runs = []
    for value in (0.5, bad):
        p, (m, v, s) = p0.clone(), _state8(n)
        now = gr.clone()
        now[7] = value
        for step in (1, 2, 3):
            sl.adamw_step([p], [now], [m], [v], step=step, scales=[s], lr=1e-2)
            now[7] = 0.5
        runs.append((p, m.view(torch.uint8), v.view(torch.uint8), *s))
    rest = torch.arange(n, device=dev()) != 7
    assert all(torch.equal(a[rest], b[rest]) for a, b in zip(runs[0][:3], runs[1][:3]))
    assert torch.equal(runs[0][3], runs[1][3]) and torch.equal(runs[0][4], runs[1][4])
    assert torch.isnan(runs[1][0][7]) and torch.isfinite(runs[0][0]).all()
