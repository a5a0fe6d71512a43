"""AdamWPlan / FusedAdamW against AdamW's formula in 64 bits, with moments in 32
and in 8 bits, over lists of dense and padded tensors.

Tolerances: m, v and p each pass at most 8 roundings to 32 bits (square root and
quotient included, 2^-24 each at most), so 8 * 2^-24 of the magnitudes added
bounds them; rounding p to its type adds half a step.  An 8-bit value is one of
the two neighbours of the exact one, a step apart: e4m3's step is at most 2^-3
of the value, or 2^-9 of the scale below its smallest normal."""
import math

import pytest
import torch

from gpu_helpers import dev

gpu = pytest.mark.gpu
U = 2.0 ** -24
HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


def _tensors(sizes, dtype, seed, sparse=()):
    g = torch.Generator().manual_seed(seed)
    ps, gs, live = [], [], []
    for k, n in enumerate(sizes):
        p, gr = torch.randn(n, generator=g), 0.1 * torch.randn(n, generator=g)
        c = None
        if k in sparse:
            c = torch.randint(-1, 4, (n,), generator=g, dtype=torch.int32)
            p[c < 0] = 0
        ps.append(p.to(dtype).to(dev()))
        gs.append(gr.to(dtype).to(dev()))
        live.append(None if c is None else c.to(dev()))
    return ps, gs, live


def _formula(p, g, m, v, step, live, lr, betas, eps, weight_decay):
    b1, b2 = betas
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    upd = lr / (1 - b1 ** step) * m1 / (v1.sqrt() / math.sqrt(1 - b2 ** step) + eps)
    p1 = p * (1 - lr * weight_decay) - upd
    if live is not None:
        on = live >= 0
        p1, m1, v1 = torch.where(on, p1, p), torch.where(on, m1, m), torch.where(on, v1, v)
    return p1, m1, v1, upd.abs()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("count", [1, 7, 49, 400])
def test_moments_in_32_bits(dtype, count):
    import sparsecore_b200 as sl

    g = torch.Generator().manual_seed(count)
    sizes = [int(n) for n in torch.randint(0, 6000, (count,), generator=g)]
    sizes[0] = 1
    ps, gs, live = _tensors(sizes, dtype, count, sparse=range(0, count, 3))
    ms, vs = [torch.zeros(n, device=dev()) for n in sizes], [torch.zeros(n, device=dev()) for n in sizes]
    plan = sl.AdamWPlan(ps, ms, vs, live=live)
    for step in (1, 2, 3):
        old = [(p.double(), m.double(), v.double()) for p, m, v in zip(ps, ms, vs)]
        plan.step(gs, step=step, **HYPER)
        for (p0, m0, v0), p, gr, m, v, c in zip(old, ps, gs, ms, vs, live):
            p1, m1, v1, upd = _formula(p0, gr.double(), m0, v0, step, c, **HYPER)
            assert bool(((m.double() - m1).abs() <= 8 * U * (m0.abs() + gr.double().abs()) + 1e-44).all())
            assert bool(((v.double() - v1).abs() <= 8 * U * v1 + 1e-44).all())
            # m may cancel: its error, over the root, is the update's
            merr = 8 * U * (m0.abs() + gr.double().abs()) / m1.abs().clamp_min(1e-30)
            lim = U * 8 * (p0.abs() + upd) + upd * merr + torch.finfo(dtype).eps / 2 * p1.abs() * 1.01 + 1e-7 * (dtype == torch.float16)
            assert bool(((p.double() - p1).abs() <= lim).all())
            if c is not None:
                assert not p[c < 0].any() and not m[c < 0].any()


def _grid():
    return torch.arange(0x7F, dtype=torch.uint8, device=dev()).view(torch.float8_e4m3fn).double()


def _neighbours(x):
    """The 8-bit values around x (0 to 448), 1e-6 of slack for the last bits of x itself; where x is an
    8-bit value to within them, that one lies between the two."""
    grid = _grid()
    lo = grid[(torch.searchsorted(grid, x * (1 - 1e-6), right=True) - 1).clamp_min(0)]
    hi = grid[torch.searchsorted(grid, x * (1 + 1e-6) - 1e-12).clamp_max(grid.numel() - 1)]
    return lo, hi


def _blocked(t):
    return torch.nn.functional.pad(t, (0, -t.numel() % 256)).view(-1, 256)


def _state8(n):
    z = lambda: torch.zeros(n, dtype=torch.uint8, device=dev()).view(torch.float8_e4m3fn)  # noqa: E731
    return z(), z(), (torch.zeros(-(-n // 256), device=dev()), torch.zeros(-(-n // 256), device=dev()))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes", [[1], [255, 256, 257], [2047, 2048, 2049, 5000, 3], [100] * 60])
def test_moments_in_8_bits(dtype, sizes):
    import sparsecore_b200 as sl

    ps, gs, live = _tensors(sizes, dtype, len(sizes), sparse=(1,))
    st = [_state8(n) for n in sizes]
    plan = sl.AdamWPlan(ps, [s[0] for s in st], [s[1] for s in st], live=live, scales=[s[2] for s in st])
    for step in (1, 2, 3):
        old = [(p.double(), (_blocked(m.double()) * s[0][:, None].double()).view(-1)[:p.numel()],
                (_blocked(v.double()) * s[1][:, None].double()).view(-1)[:p.numel()] ** 2) for p, (m, v, s) in zip(ps, st)]
        plan.step(gs, step=step, seed=5, **HYPER)
        for (p0, m0, v0), p, gr, (m, v, s), c in zip(old, ps, gs, st, live):
            n = p.numel()
            p1, m1, v1, upd = _formula(p0, gr.double(), m0, v0, step, c, **HYPER)
            merr = 16 * U * (m0.abs() + gr.double().abs()) / m1.abs().clamp_min(1e-30)
            lim = U * 16 * (p0.abs() + upd) + upd * merr + torch.finfo(dtype).eps / 2 * p1.abs() * 1.01 + 1e-7 * (dtype == torch.float16)
            assert bool(((p.double() - p1).abs() <= lim).all())
            for val, held, scale in ((m1, m, s[0]), (v1.sqrt(), v, s[1])):
                top = _blocked(val.abs()).amax(1).clamp_min(2.0 ** -100)
                torch.testing.assert_close(scale.double(), top / 448, rtol=1e-6, atol=0)
                x = (_blocked(val.abs()) / top[:, None] * 448).view(-1)[:n]
                lo, hi = _neighbours(x.clamp_max(448))
                q = held.double().abs()
                ok = (q >= lo) & (q <= hi)
                if held is v:  # a root above zero is not held as zero
                    ok |= (val > 0) & (q == 2.0 ** -9) & (x < 2.0 ** -9)
                    assert bool((q[val > 0] > 0).all())
                assert bool(ok.all())
                assert bool(((held.double() * val) >= 0).all())


def _mixed(v):
    for shift, factor in ((16, 0x5B2C9E6D), (13, 0x3F4A7C15)):
        v = (v ^ (v >> shift)) * factor & 0xFFFFFFFF
    return v ^ (v >> 16)


def _cut(val, bits, keep):
    """Values over their block's scale, up or down by 16 bits, in 32-bit operations."""
    b = _blocked(val)
    top = b.abs().amax(1, keepdim=True).clamp_min(2.0 ** -100)
    x = (b.abs() * (448.0 / top)).clamp_max(448.0)
    low = torch.where(x < 2.0 ** -6, 2.0 ** -6, 0.0).float()
    q = (((x + low).view(torch.int32) + (_blocked(bits).to(torch.int32) << 4)) & ~0xFFFFF).view(torch.float32) - low
    if keep:
        q = torch.where(b > 0, q.clamp_min(2.0 ** -9), q)
    q = torch.where(b < 0, -q, q)
    return q.to(torch.float8_e4m3fn).view(-1)[:val.numel()], (top * (1.0 / 448.0))[:, 0]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_8_bit_moments_are_the_formulas_bit_for_bit(dtype):
    """Each operation of the formula rounded to 32 bits by itself gives the held bytes and scales
    exactly, step after step: what is held does not depend on how the kernel groups its work."""
    import sparsecore_b200 as sl

    sizes = [70000, 2048, 300, 1]
    ps, gs, live = _tensors(sizes, dtype, 11, sparse=(2,))
    st = [_state8(n) for n in sizes]
    b1, b2 = HYPER["betas"]
    ref = [[m.clone(), v.clone(), (s[0].clone(), s[1].clone())] for m, v, s in st]
    for step in range(1, 6):
        gs = [g * (1 + 0.3 * step) for g in gs]
        sl.adamw_step(ps, gs, [s[0] for s in st], [s[1] for s in st], step=step, live=live, scales=[s[2] for s in st], seed=9, **HYPER)
        for i, (g, c, r, n) in enumerate(zip(gs, live, ref, sizes)):
            mf = (_blocked(r[0].float()) * r[2][0][:, None]).view(-1)[:n]
            vf = (_blocked(r[1].float()) * r[2][1][:, None]).view(-1)[:n].square()
            gf = g.float()
            m1 = mf + (gf - mf) * (1 - b1)
            v1 = vf * b2 + gf * gf * (1 - b2)
            root = v1.sqrt()
            if c is not None:
                held = (_blocked(r[1].float()) * r[2][1][:, None]).view(-1)[:n]
                m1, root = torch.where(c < 0, mf, m1), torch.where(c < 0, held, root)
            key = _mixed((9 + 0x9E3779B1 * step + 0x85EBCA77 * i) & 0xFFFFFFFF)
            bits = _mixed((torch.arange(n, device=dev()) * 0x9E3779B1 + key) & 0xFFFFFFFF)
            r[0], sm = _cut(m1, bits & 0xFFFF, False)
            r[1], sv = _cut(root, bits >> 16, True)
            r[2] = (sm, sv)
            m, v, s = st[i]
            assert torch.equal(m.view(torch.uint8), r[0].view(torch.uint8)) and torch.equal(v.view(torch.uint8), r[1].view(torch.uint8))
            assert torch.equal(s[0], sm) and torch.equal(s[1], sv)


@gpu
def test_8_bit_values_are_right_on_average():
    """1000 times the same moments under other seeds: the mean of the held values
    approaches the exact ones as the dither's deviation over sqrt(1000).  A value
    between neighbours a step apart has a deviation of at most half a step, 2^-4 of
    it; five deviations of the mean, 5 / sqrt(1000) * 2^-4 = 0.0099, hold for
    each of 512 values but for one run in 3000."""
    import sparsecore_b200 as sl

    n = 512
    g = torch.Generator().manual_seed(3)
    gr = (0.5 + torch.rand(n, generator=g)).to(dev())
    total = torch.zeros(2, n, dtype=torch.float64, device=dev())
    for seed in range(1000):
        p, (m, v, s) = torch.zeros(n, device=dev()), _state8(n)
        sl.adamw_step([p], [gr], [m], [v], step=1, scales=[s], seed=seed, **HYPER)
        total[0] += (_blocked(m.double()) * s[0][:, None]).view(-1)
        total[1] += (_blocked(v.double()) * s[1][:, None]).view(-1)
    m1, r1 = 0.1 * gr.double(), (0.01 * gr.double() ** 2).sqrt()
    for mean, exact in ((total[0] / 1000, m1), (total[1] / 1000, r1)):
        assert float(((mean - exact) / exact).abs().max()) < 0.0099


@gpu
def test_what_is_not_finite_spoils_no_neighbour():
    import sparsecore_b200 as sl

    n = 300
    for bad in (float("nan"), float("inf")):
        a, b = [], []
        for out in (a, b):
            ps, gs, _ = _tensors([n], torch.float32, 1)
            m, v, s = _state8(n)
            if out is b:
                gs[0][7] = bad
            for step in (1, 2):
                sl.adamw_step(ps, gs, [m], [v], step=step, scales=[s], **HYPER)
            out += [ps[0], m.float(), v.float(), s[0]]
        rest = torch.arange(n, device=dev()) != 7
        assert torch.isnan(b[0][7]) and torch.isnan(b[1][7]) and torch.isnan(b[2][7])
        assert torch.isfinite(b[0][rest]).all() and torch.isfinite(b[3]).all()
        if gs[0][rest].abs().max() > 0 and torch.equal(a[3], b[3]):  # element 7 was not its block's largest
            assert torch.equal(a[0][rest], b[0][rest])


@gpu
def test_no_gradient_for_a_while_does_not_blow_up():
    """Elements whose gradient stays zero after one small one: the root's 8-bit
    value must not reach zero before the first moment's does."""
    import sparsecore_b200 as sl

    n = 256
    p, (m, v, s) = torch.zeros(n, device=dev()), _state8(n)
    gr = torch.full((n,), 1e-4, device=dev())
    gr[0] = 100.0
    for step in range(1, 40):
        before = p.clone()
        sl.adamw_step([p], [gr], [m], [v], step=step, scales=[s], seed=step, lr=1e-3, weight_decay=0.0)
        assert float((p - before).abs().max()) <= 0.02  # 1e-3 * m / root: the two are held a few steps apart at most
        gr[1:] = 0


@gpu
def test_unaligned_tensors_and_missing_gradients():
    import sparsecore_b200 as sl

    for bits in (32, 8):
        base = torch.randn(4, 3001, device=dev())
        p, gr = base[0][1:2500], base[1][3:2502]
        n = p.numel()
        q = p.clone()
        if bits == 32:
            st, st2 = [torch.zeros(n + 1, device=dev())[1:] for _ in range(2)], [torch.zeros(n, device=dev()) for _ in range(2)]
            sc = sc2 = None
        else:
            a, b = _state8(n), _state8(n)
            st = [torch.zeros(n + 3, dtype=torch.uint8, device=dev())[3:].view(torch.float8_e4m3fn) for _ in range(2)]
            st2, sc, sc2 = list(b[:2]), [a[2]], [b[2]]
        guard = base.clone()
        sl.adamw_step([p], [gr], st[:1], st[1:], step=1, scales=sc, **HYPER)
        sl.adamw_step([q], [gr.clone()], st2[:1], st2[1:], step=1, scales=sc2, **HYPER)
        assert torch.equal(p, q) and torch.equal(st[0].float(), st2[0].float())
        assert torch.equal(base[0][2500:], guard[0][2500:]) and base[0][0] == guard[0][0] and torch.equal(base[1:], guard[1:])
    ps, gs, _ = _tensors([10, 20, 30], torch.float32, 2)
    ms, vs = [torch.zeros_like(p) for p in ps], [torch.zeros_like(p) for p in ps]
    keep = [p.clone() for p in ps]
    sl.adamw_step(ps, [gs[0], None, gs[2]], ms, vs, step=1, **HYPER)
    assert torch.equal(ps[1], keep[1]) and not torch.equal(ps[0], keep[0]) and not torch.equal(ps[2], keep[2])
    sl.adamw_step(ps, [None] * 3, ms, vs, step=1, **HYPER)
    sl.adamw_step([], [], [], [], step=1)


def _model(seed=3):
    import sparsecore_b200 as sl

    torch.manual_seed(seed)
    return torch.nn.Sequential(sl.SparseLinear(96, 64, sparsity=0.8, device=dev()), torch.nn.GELU(),
                               sl.SparseLinear(64, 32, sparsity=0.9, device=dev()), torch.nn.Linear(32, 8).to(dev()))


@gpu
def test_fused_adamw_follows_torch_across_a_topology_update():
    import sparsecore_b200 as sl

    a, b = _model(), _model()
    opt_a = torch.optim.AdamW(a.parameters(), lr=3e-3, weight_decay=0.01)
    opt_b = sl.FusedAdamW(b, lr=3e-3, weight_decay=0.01)
    algos = [sl.SET(0.8, drop_fraction=0.3, update_freq=4, seed=1) for _ in range(2)]
    a.apply(algos[0])
    b.apply(algos[1])
    g = torch.Generator().manual_seed(0)
    for _ in range(9):
        x = torch.randn(40, 96, generator=g).to(dev())
        for model, opt, algo in ((a, opt_a, algos[0]), (b, opt_b, algos[1])):
            opt.zero_grad(set_to_none=True)
            model(x).square().mean().backward()
            opt.step()
            algo.step()
        for m_a, m_b in zip(a, b):
            if isinstance(m_a, sl.SparseLinear):
                assert torch.equal(m_a._csr.col_indices, m_b._csr.col_indices)
                torch.testing.assert_close(m_b._values, m_a._values, rtol=1e-5, atol=1e-7)
                assert not m_b._values[m_b._csr.col_indices < 0].any()
    torch.testing.assert_close(b[3].weight, a[3].weight, rtol=1e-5, atol=1e-7)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_equal_eager_ones(bits):
    import sparsecore_b200 as sl

    models = [_model(), _model()]
    opts = [sl.FusedAdamW(m, lr=torch.tensor(3e-3, device=dev()), capturable=True, state_bits=bits) for m in models]
    x = torch.randn(40, 96, device=dev())

    def once(k):
        opts[k].zero_grad(set_to_none=True)
        models[k](x).square().mean().backward()
        opts[k].step()

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        once(0)
        once(1)
    torch.cuda.current_stream().wait_stream(s)
    opts[0].zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        once(0)
    for k in range(4):
        if k == 2:
            for o in opts:
                o.param_groups[0]["lr"].mul_(0.1)
        graph.replay()
        once(1)
    torch.cuda.synchronize()
    assert int(opts[0].param_groups[0]["step"]) == 5
    for p, q in zip(models[0].parameters(), models[1].parameters()):
        assert torch.equal(p, q)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_state_goes_through_a_checkpoint(bits):
    import sparsecore_b200 as sl

    a, b = _model(), _model()
    kw = dict(lr=3e-3, state_bits=bits)
    oa, ob = sl.FusedAdamW(a, **kw), sl.FusedAdamW(b, **kw)
    x = torch.randn(40, 96, device=dev())

    def once(m, o):
        o.zero_grad()
        m(x).square().mean().backward()
        o.step()

    once(a, oa)
    b.load_state_dict(a.state_dict())
    ob.load_state_dict(oa.state_dict())
    once(a, oa)
    once(b, ob)
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p, q)
        for u, w in zip(oa.state_values(p), ob.state_values(q)):
            assert u.shape == p.shape and torch.equal(u, w)


@gpu
def test_a_layer_drawn_again_and_a_state_of_other_bits():
    import sparsecore_b200 as sl

    model, x = _model(), torch.randn(40, 96, device=dev())
    opts = {bits: sl.FusedAdamW(model, state_bits=bits) for bits in (32, 8)}
    for _ in range(2):
        for o in opts.values():
            o.zero_grad()
            model(x).square().mean().backward()
            o.step()
        model[0].reset_parameters()  # another mask: another number of slots
    assert torch.isfinite(model(x)).all() and not model[0]._values[model[0]._csr.col_indices < 0].any()
    for a, b in ((32, 8), (8, 32)):
        with pytest.raises(ValueError):
            opts[a].load_state_dict(opts[b].state_dict())


def test_refusals_without_a_gpu():
    import sparsecore_b200 as sl

    p = torch.zeros(4)
    with pytest.raises(RuntimeError, match="CUDA"):
        sl.adamw_step([p], [p], [p], [p], step=1)
    with pytest.raises(ValueError):
        sl.AdamWPlan([p], [], [p])
    lin = torch.nn.Linear(2, 2)
    for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(state_bits=4), dict(lr=torch.tensor(1e-3))):
        with pytest.raises(ValueError):
            sl.FusedAdamW(lin, **kw)


@gpu
def test_refusals():
    import sparsecore_b200 as sl

    z = lambda n=8, **k: torch.zeros(n, device=dev(), **k)  # noqa: E731
    good = dict(params=[z()], grads=[z()], exp_avgs=[z()], exp_avg_sqs=[z()], step=1)
    shared = z(16)
    for kw in (dict(step=0), dict(lr=-1.0), dict(grads=[z(7)]), dict(grads=[z().half()]), dict(exp_avgs=[z(7)]),
               dict(exp_avgs=[z().half()]), dict(params=[z().double()]), dict(live=[z()]), dict(grads=[]),
               dict(scales=[(z(1), z(1))]), dict(params=[z(16)[::2]]), dict(params=[shared[:8]], exp_avgs=[shared[4:12]])):
        with pytest.raises(ValueError):
            sl.adamw_step(**(good | kw))
    with pytest.raises(RuntimeError):
        sl.adamw_step(**(good | dict(grads=[torch.zeros(8)])))
    with pytest.raises(TypeError):
        sl.adamw_step(**(good | dict(exp_avgs=[1])))
