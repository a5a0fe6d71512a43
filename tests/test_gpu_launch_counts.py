"""The launches that the package counts for its fused training operators are
the kernel nodes of a captured call."""
import pytest
import torch

from gpu_helpers import dev

gpu = pytest.mark.gpu


def _nodes(fn):
    """(kernel nodes of the graph that `fn` captures to, launches counted meanwhile)."""
    runtime = pytest.importorskip("cuda.bindings.runtime")
    from sparsecore_b200 import _native as N

    fn()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        before = N.launches["count"]
        fn()
        counted = N.launches["count"] - before
    err, _, n = runtime.cudaGraphGetNodes(graph.raw_cuda_graph())
    err, nodes, n = runtime.cudaGraphGetNodes(graph.raw_cuda_graph(), n)
    kinds = [runtime.cudaGraphNodeGetType(q)[1] for q in nodes[:n]]
    return sum(k == runtime.cudaGraphNodeType.cudaGraphNodeTypeKernel for k in kinds), counted


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,D,V", [(300, 64, 100), (300, 72, 1000), (16384, 384, 65), (20000, 40, 7000)])
def test_loss(T, D, V, dtype):
    import sparsecore_b200 as sl

    x, w = torch.randn(T, D, device=dev()).to(dtype), torch.randn(V, D, device=dev()).to(dtype)
    t = torch.randint(0, V, (T,), device=dev())
    real, counted = _nodes(lambda: sl.linear_cross_entropy(x, w, t))
    assert counted == real and real >= 1
    xl, wl, one = x.requires_grad_(), w.requires_grad_(), torch.ones((), device=dev())
    for wanted in ((xl, wl), (xl,)):
        real, counted = _nodes(lambda: torch.autograd.grad(sl.linear_cross_entropy(xl, wl, t), wanted, one))
        assert counted == real and real >= 3


@gpu
@pytest.mark.parametrize("post", [False, True])
def test_norm(post):
    import sparsecore_b200 as sl

    y, r = (torch.randn(300, 96, device=dev(), requires_grad=True) for _ in range(2))
    w = torch.ones(96, device=dev())
    g = torch.ones(300, 96, device=dev())
    for vectors in (False, True):
        wl = w.clone().requires_grad_(vectors)
        pw = w.clone().requires_grad_(vectors) if post else None

        def once():
            out, h = sl.residual_norm(y, r, wl, post_weight=pw)
            torch.autograd.grad((out, h), [t for t in (y, r, wl, pw) if t is not None and t.requires_grad], (g, g))

        real, counted = _nodes(once)
        assert counted == real == 2 + vectors


@gpu
@pytest.mark.parametrize("count", [1, 400, 1000])
def test_adamw(count):
    import sparsecore_b200 as sl

    make = lambda: [torch.zeros(8, device=dev()) for _ in range(count)]  # noqa: E731
    ps, gs, ms, vs = make(), make(), make(), make()
    plan = sl.AdamWPlan(ps, ms, vs)
    real, counted = _nodes(lambda: plan.step(gs, step=1))
    assert counted == real == -(-count // 384)
