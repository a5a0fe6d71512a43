"""residual_norm against its formula in 64 bits: values, every gradient, the
types, widths and gates where it can go wrong, and graph replay.

Tolerances are bounds by arithmetic.  Every quantity is a chain of at most 16
roundings to 32 bits and of sums over at most 32 values a thread, 16 warps and
five shuffles, each off by at most 2^-24 of the sum of the magnitudes it adds:
64 * 2^-24 of those magnitudes covers them.  Rounding to the output's type
adds half a step, eps / 2 of the value."""
import pytest
import torch

from gpu_helpers import dev

gpu = pytest.mark.gpu
U = 2.0 ** -24


def _within(got, ref, mag, k=64):
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    d = (got.double() - ref).abs()
    lim = k * U * mag + half * (ref.abs() + k * U * mag) + tiny
    assert bool((d <= lim).all()), f"off by {float((d / lim).max()):.3g} times the bound"


def _case(T, D, dtype, seed, kind="layer", post=False, gate=None, rdtype=None, wdtype=None, offset=0.3, bias=True):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    wd, rd = wdtype or dtype, rdtype or dtype
    c = {"y": rn(T, D).to(dtype), "r": (2 * rn(T, D) + offset).to(rd), "w": (1 + 0.1 * rn(D)).to(wd),
         "b": (0.1 * rn(D)).to(wd) if bias else None, "gate": None, "pw": None, "pb": None,
         "dout": rn(T, D).to(rd), "dh": rn(T, D).to(dtype)}
    if gate is not None:
        c["gate"] = rn(*gate, D).to(wd)
    if post:
        c["pw"], c["pb"] = (1 + 0.1 * rn(D)).to(wd), (0.1 * rn(D)).to(wd) if bias else None
    return {k: None if v is None else v.to(dev()) for k, v in c.items()} | {"kind": kind}


def _norm64(v, w, b, kind, eps):
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
    rstd = 1 / torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + eps)
    n = (v - mean) * rstd
    return n * w + (0 if b is None else b), n, mean, rstd


def _spread(gate, T):
    return gate.repeat_interleave(T // gate.shape[0], 0)


def _check(c, scale=0.7, eps=1e-5, grads=True, learned=True):
    import sparsecore_b200 as sl

    names = [k for k in ("y", "r", "w", "b", "gate", "pw", "pb") if c[k] is not None]
    leaf = {k: c[k].clone().requires_grad_(grads) for k in names}
    st = torch.full((1,), scale, device=dev(), requires_grad=grads) if learned else scale
    gate, y, r = leaf.get("gate"), leaf["y"], leaf["r"]
    if gate is not None and gate.shape[0] != y.shape[0]:  # a gate per sequence, of as many equal sequences
        G = gate.shape[0]
        y, r, gate = y.view(G, -1, y.shape[1]), r.view(G, -1, r.shape[1]), gate[:, None] if G > 1 else gate[0]
    out, h = sl.residual_norm(y, r, leaf["w"], leaf.get("b"), kind=c["kind"], eps=eps, gate=gate, scale=st,
                              post_weight=leaf.get("pw"), post_bias=leaf.get("pb"))
    out, h = out.view(leaf["y"].shape), h.view(leaf["y"].shape)
    assert out.dtype == c["r"].dtype and h.dtype == c["y"].dtype
    a = {k: c[k].double() for k in names}
    T, D = a["y"].shape
    if learned:
        scale = float(st.detach())  # as held in 32 bits
    pn = pmag = torch.zeros_like(a["y"])
    u, umag, prstd = a["y"], a["y"].abs(), None
    if "pw" in a:
        u, pn, pmean, prstd = _norm64(a["y"], a["pw"], a.get("pb"), c["kind"], eps)
        pmag = pn.abs() + 1 + pmean.abs() * prstd
        umag = u.abs() + a["pw"].abs() * pmag
    ga = _spread(a["gate"], T) if "gate" in a else torch.ones_like(u)
    ref = a["r"] + scale * ga * u
    _within(out, ref, a["r"].abs() + scale * ga.abs() * umag)
    held = out.detach().double()  # the norm is of the stream as it is held
    href, n, mean, rstd = _norm64(held, a["w"], a.get("b"), c["kind"], eps)
    nmag = n.abs() + 1 + mean.abs() * rstd
    _within(h, href, href.abs() + a["w"].abs() * nmag)
    if not grads:
        return
    named = {k: leaf[k] for k in names} | ({"scale": st} if learned else {})
    got = dict(zip(named, torch.autograd.grad((out, h), list(named.values()), (c["dout"], c["dh"]))))
    do, dh = c["dout"].double(), c["dh"].double()

    def back(d, dmag, n, nmag, w, rstd):
        dn, m = d * w, dmag * w.abs()
        v = dn - n * (dn * n).mean(-1, keepdim=True)
        mag = m + nmag * (m * nmag).mean(-1, keepdim=True)
        if c["kind"] == "layer":
            v, mag = v - dn.mean(-1, keepdim=True), mag + m.mean(-1, keepdim=True)
        return v * rstd, mag * rstd

    v, m = back(dh, dh.abs(), n, nmag, a["w"], rstd)
    d, dmag = do + v, do.abs() + m
    _within(got["r"], d, dmag)
    rows = 64 + T  # a column's sum is at most T long
    _within(got["w"], (dh * n).sum(0), (dh.abs() * nmag).sum(0), rows)
    if "b" in a:
        _within(got["b"], dh.sum(0), dh.abs().sum(0), rows)
    if learned:
        _within(got["scale"], (d * ga * u).sum().reshape(1), (dmag * ga.abs() * umag).sum().reshape(1), 64 + T + D)
    du, dumag = scale * d, scale * dmag
    if "gate" in a:
        G = a["gate"].shape[0]
        _within(got["gate"], (du * u).view(G, -1, D).sum(1), (dumag * umag).view(G, -1, D).sum(1), rows)
    du, dumag = du * ga, dumag * ga.abs()
    if "pw" in a:
        _within(got["pw"], (du * pn).sum(0), (dumag * pmag).sum(0), rows)
        if "pb" in a:
            _within(got["pb"], du.sum(0), dumag.sum(0), rows)
        du, dumag = back(du, dumag, pn, pmag, a["pw"], prstd)
    _within(got["y"], du, dumag)


@gpu
@pytest.mark.parametrize("D", [1, 3, 31, 64, 257, 768, 2048, 2052, 4096, 5000, 8192, 16384, 16383])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_widths(D, dtype):
    _check(_case(5, D, dtype, D, kind="rms" if D % 2 else "layer", post=D % 3 == 0, gate=(1,)))


@gpu
@pytest.mark.parametrize("D", [1, 5, 32, 96, 200, 384, 513, 768, 1000, 1024, 1280, 2048, 2500, 4096, 6000, 8192, 16384])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [3, 1337])
def test_a_plain_residual_and_norm(D, dtype, T):
    """Nothing after the block: the pass back that most models take, at every width it is spread differently."""
    c = _case(T, D, dtype, D + T, kind="rms" if D % 5 == 0 else "layer")
    _check(c, scale=1.0, learned=False)
    if T == 3:
        _check(c, scale=0.5, learned=False)


@gpu
@pytest.mark.parametrize("T", [1, 2, 147, 1185, 5001])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_rows(T, post, kind):
    _check(_case(T, 384, torch.float32, T, kind=kind, post=post))


@gpu
@pytest.mark.parametrize("groups", [1, 2, 6, 40, 600, 1200])
@pytest.mark.parametrize("D", [96, 50])
@pytest.mark.parametrize("post", [True, False])
def test_gates_shared_by_runs_of_rows(groups, D, post):
    c = _case(1200, D, torch.float32, groups, gate=(groups,), post=post)
    _check(c)
    _check(c, scale=0.5, learned=False)
    _check({k: v.bfloat16() if torch.is_tensor(v) else v for k, v in c.items()} | {"kind": "rms"})


@gpu
@pytest.mark.parametrize("groups", [1, 4, 600, 1200])
def test_a_gate_that_asks_for_no_gradient(groups):
    """Then a CTA's rows may cross from one sequence's gate to the next."""
    import sparsecore_b200 as sl

    c = _case(1200, 96, torch.float32, groups + 7, gate=(groups,))
    y, r, w = (c[k].clone().requires_grad_() for k in ("y", "r", "w"))
    S = 1200 // groups
    gate = c["gate"][:, None] if groups > 1 else c["gate"][0]
    out, h = sl.residual_norm(y.view(groups, S, 96), r.view(groups, S, 96), w, gate=gate, kind="rms")
    gy, gr, gw = torch.autograd.grad((out, h), (y, r, w), (c["dout"].view(groups, S, 96), c["dh"].view(groups, S, 96)))
    _within(gy, gr.double() * _spread(c["gate"].double(), 1200), gr.double().abs() * _spread(c["gate"].double(), 1200).abs())


@gpu
@pytest.mark.parametrize("rdtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("wdtype", [torch.bfloat16, torch.float32])
def test_mixed_types(rdtype, wdtype):
    _check(_case(333, 512, torch.bfloat16, 5, rdtype=rdtype, wdtype=wdtype, gate=(333,), post=True))


@gpu
def test_without_bias_and_far_means():
    _check(_case(64, 768, torch.float32, 1, bias=False, post=True))
    _check(_case(64, 768, torch.float32, 2, offset=300.0))
    _check(_case(64, 768, torch.float32, 3), grads=False)


@gpu
def test_orders_and_strides():
    """Slices, transposed operands and bases off the vector width."""
    c = _case(40, 200, torch.float32, 4)
    base = torch.randn(200, 40, device=dev())
    c["y"] = base.t()
    c["r"] = torch.randn(40, 201, device=dev())[:, 1:]
    c["w"] = torch.randn(201, device=dev())[1:]
    _check(c)


@gpu
def test_leading_dimensions_and_a_gate_per_sequence():
    import sparsecore_b200 as sl

    y, r = torch.randn(3, 7, 64, device=dev()), torch.randn(3, 7, 64, device=dev())
    w, gate = torch.randn(64, device=dev()), torch.randn(3, 1, 64, device=dev())
    out, h = sl.residual_norm(y, r, w, gate=gate, kind="rms")
    assert out.shape == h.shape == y.shape
    flat, hf = sl.residual_norm(y.view(21, 64), r.view(21, 64), w, gate=gate.repeat_interleave(7, 0).view(21, 64), kind="rms")
    assert torch.equal(out.view(21, 64), flat) and torch.equal(h.view(21, 64), hf)
    with pytest.raises(ValueError):  # [3, 64] would be a gate per position to some, per sequence to others
        sl.residual_norm(y, r, w, gate=gate[:, 0], kind="rms")


@gpu
@pytest.mark.parametrize("use", ["out", "h"])
def test_only_one_output_is_used(use):
    import sparsecore_b200 as sl

    c = _case(33, 96, torch.float32, 8)
    y, r, w, b = (c[k].clone().requires_grad_() for k in ("y", "r", "w", "b"))
    out, h = sl.residual_norm(y, r, w, b)
    gy, gr, gw, gb = torch.autograd.grad(out if use == "out" else h, (y, r, w, b), c["dh"])
    assert torch.equal(gy, gr)
    if use == "out":
        assert torch.equal(gr, c["dh"]) and not gw.any() and not gb.any()
    else:
        ref = torch.nn.functional.layer_norm((c["y"] + c["r"]).double().requires_grad_(), (96,), c["w"].double(), c["b"].double())
        assert torch.isfinite(gr).all() and ref.shape == h.shape and gb.abs().sum() > 0


@gpu
def test_gradients_against_differences():
    """Along one direction in all operands at once: the formula in 64 bits is
    differenced at +-1e-5, good to 1e-8 of the terms' magnitudes."""
    import sparsecore_b200 as sl

    c = _case(20, 48, torch.float32, 9, post=True, gate=(20,))
    names = ("y", "r", "w", "b", "gate", "pw", "pb")
    leaf = {k: c[k].clone().requires_grad_() for k in names}
    out, h = sl.residual_norm(leaf["y"], leaf["r"], leaf["w"], leaf["b"], gate=leaf["gate"], scale=0.7,
                              post_weight=leaf["pw"], post_bias=leaf["pb"])
    grads = torch.autograd.grad((out, h), [leaf[k] for k in names], (c["dout"], c["dh"]))
    g = torch.Generator(device=dev()).manual_seed(1)
    way = {k: torch.randn(c[k].shape, generator=g, device=dev()).double() for k in names}

    def f(e):
        a = {k: c[k].double() + e * way[k] for k in names}
        o = a["r"] + 0.7 * a["gate"] * _norm64(a["y"], a["pw"], a["pb"], "layer", 1e-5)[0]
        return (o * c["dout"]).sum() + (_norm64(o, a["w"], a["b"], "layer", 1e-5)[0] * c["dh"]).sum()

    slope = (f(1e-5) - f(-1e-5)) / 2e-5
    terms = [(gr.double() * way[k]) for gr, k in zip(grads, names)]
    total, mag = sum(t.sum() for t in terms), sum(t.abs().sum() for t in terms)
    assert abs(float(total - slope)) <= float(mag) * (256 * U + 1e-7)


@gpu
def test_rows_that_are_not_finite_stay_apart():
    import sparsecore_b200 as sl

    c = _case(9, 64, torch.float32, 10)
    clean = sl.residual_norm(c["y"], c["r"], c["w"], c["b"])
    c["y"][4, 3] = float("nan")
    c["r"][7, 0] = float("inf")
    out, h = sl.residual_norm(c["y"], c["r"], c["w"], c["b"])
    rest = [0, 1, 2, 3, 5, 6, 8]
    assert torch.equal(out[rest], clean[0][rest]) and torch.equal(h[rest], clean[1][rest])
    assert torch.isnan(h[4]).all() and torch.isnan(h[7]).any()


@gpu
def test_no_rows():
    import sparsecore_b200 as sl

    y, r = (torch.randn(0, 32, device=dev(), requires_grad=True) for _ in range(2))
    w = torch.ones(32, device=dev(), requires_grad=True)
    out, h = sl.residual_norm(y, r, w)
    (out.sum() + h.sum()).backward()
    assert out.shape == (0, 32) and y.grad.shape == (0, 32) and not w.grad.any()


@gpu
def test_runs_are_repeatable_and_replay_in_a_graph():
    import sparsecore_b200 as sl

    c = _case(300, 768, torch.float32, 11, post=True, gate=(1,))
    names = ("y", "r", "w", "b", "gate", "pw", "pb")
    leaf = {k: c[k].clone().requires_grad_() for k in names}

    def once():
        out, h = sl.residual_norm(leaf["y"], leaf["r"], leaf["w"], leaf["b"], gate=leaf["gate"], scale=0.5,
                                  post_weight=leaf["pw"], post_bias=leaf["pb"])
        return [out.detach(), h.detach(), *torch.autograd.grad((out, h), [leaf[k] for k in names], (c["dout"], c["dh"]))]

    first, second = once(), once()
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        once()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once()
    with torch.no_grad():
        leaf["y"].mul_(0.5)
    want = once()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, want))


@gpu
def test_second_derivatives_are_refused():
    """The gradients are not differentiable again, and say so."""
    import sparsecore_b200 as sl

    y, w = torch.randn(4, 8, device=dev(), requires_grad=True), torch.ones(8, device=dev(), requires_grad=True)
    t = torch.zeros(4, dtype=torch.int64, device=dev())
    for out in (sl.residual_norm(y, y.detach(), w)[1].square().sum(), sl.linear_cross_entropy(y, w.expand(5, 8), t)):
        (g,) = torch.autograd.grad(out, (y,), create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()


def test_refusals():
    import sparsecore_b200 as sl

    y, w = torch.zeros(4, 8), torch.ones(8)
    with pytest.raises(TypeError):
        sl.residual_norm([1.0], y, w)
    with pytest.raises(ValueError, match="kind"):
        sl.residual_norm(y, y, w, kind="batch")
    with pytest.raises(RuntimeError, match="CUDA"):
        sl.residual_norm(y, y, w)


@gpu
def test_refusals_of_shapes_and_types():
    import sparsecore_b200 as sl

    y, w = torch.zeros(4, 8, device=dev()), torch.ones(8, device=dev())
    for kw in (dict(weight=w[:4]), dict(residual=y[:2]), dict(weight=w.half()), dict(residual=y.half()), dict(y=y.double()),
               dict(gate=torch.ones(3, 8, device=dev())), dict(gate=torch.ones(8, 4, device=dev())), dict(post_bias=w),
               dict(scale=torch.ones(2, device=dev())), dict(eps=-1.0), dict(bias=torch.ones(8, 1, device=dev())),
               dict(y=torch.zeros(2, 16385, device=dev()), residual=torch.zeros(2, 16385, device=dev()))):
        with pytest.raises(ValueError):
            sl.residual_norm(**(dict(y=y, residual=y, weight=w) | kw))
    with pytest.raises(RuntimeError):
        sl.residual_norm(y, y, w.cpu())
