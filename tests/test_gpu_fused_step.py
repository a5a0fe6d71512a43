"""A whole training step on the fused operators (MiniGPT(fused=True), lm_loss,
FusedAdamW): gradients against the unfused model's, eager against captured
steps over a topology update, and 16-bit copies of the parts together.

Gradients of the two models differ by roundings alone.  Two blocks are about
40 operations in a row, forward and backward, each off by at most 64 * 2^-24
of its operands' norms: 80 * 64 * 2^-24 = 3.1e-4 of a gradient's norm bounds
what they add up to."""
import dataclasses

import pytest
import torch

from gpu_helpers import dev

pytestmark = pytest.mark.gpu
BOUND = 80 * 64 * 2.0 ** -24


def _cfg(name, **kw):
    from sparsecore_b200 import workloads as W

    return dataclasses.replace(W.CFG4 if name == "cfg4" else W.CFG5, n_layers=2, batch=4, **kw)


def _model(cfg, fused):
    from sparsecore_b200.workloads import MiniGPT

    torch.manual_seed(0)
    return MiniGPT(cfg, device=dev(), fused=fused)


@pytest.mark.parametrize("name", ["cfg4", "cfg5"])
def test_gradients_equal_the_unfused_models(name):
    from sparsecore_b200.workloads import lm_loss, synthetic_tokens

    cfg = _cfg(name)
    tok = synthetic_tokens(cfg, cfg.batch, seed=5).to(dev())
    a, b = _model(cfg, False), _model(cfg, True)
    la, lb = lm_loss(a, tok), lm_loss(b, tok)
    assert abs(float(la.detach()) - float(lb.detach())) <= BOUND * abs(float(la.detach()))
    la.backward()
    lb.backward()
    pa, pb = dict(a.named_parameters()), dict(b.named_parameters())
    assert pa.keys() == pb.keys()
    for k in pa:
        assert torch.equal(pa[k], pb[k]), k
        ga, gb = pa[k].grad.double(), pb[k].grad.double()
        assert float((ga - gb).norm()) <= BOUND * float(ga.norm()), k
    with torch.no_grad():
        assert b(tok[:, :-1]).shape == (cfg.batch, cfg.seq_len, cfg.vocab)


def _steps(cfg, graph, bits, n=7):
    import sparsecore_b200 as sl
    from sparsecore_b200.graph import GraphedStep
    from sparsecore_b200.workloads import lm_loss, synthetic_tokens

    model = _model(cfg, True)
    algo = sl.SET(sparsity=cfg.ffn_sparsity, drop_fraction=0.3, update_freq=3, seed=0)
    model.apply(algo)
    opt = sl.FusedAdamW(model, lr=cfg.lr, capturable=True, state_bits=bits)
    tok = synthetic_tokens(cfg, cfg.batch, seed=5).to(dev())

    def train(t):
        opt.zero_grad(set_to_none=True)
        loss = lm_loss(model, t)
        loss.backward()
        opt.step()
        return loss

    losses = [float(train(tok).detach())]
    algo.step()
    gs = GraphedStep(model, train, (tok,)) if graph else None
    for _ in range(n - 1):
        losses.append(float((gs() if graph else train(tok)).detach()))
        algo.step()
    for m in model.modules():
        if isinstance(m, sl.SparseLinear):
            m._csr.assert_invariants()
            assert not m._values[m._csr.col_indices < 0].any()
    return losses, [p.detach().clone() for p in model.parameters()]


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_equal_eager_ones_over_topology_updates(bits):
    """Config 4's sizes: every operation of its step is deterministic."""
    cfg = _cfg("cfg4")
    eager, pe = _steps(cfg, False, bits)
    again, pa = _steps(cfg, False, bits)
    graphed, pg = _steps(cfg, True, bits)
    assert eager == again == graphed
    assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(pe, pa, pg))
    assert all(torch.isfinite(torch.tensor(eager)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_norm_loss_and_step_in_16_bits(dtype):
    """Residual block, head, loss and one AdamW step on 16-bit tensors, in a row and
    from one backward pass; against the same in 64 bits from the rounded outputs.

    Held values are off by eps / 2 each; the gradient of the block's output passes
    three such roundings (loss, norm, its own), the others two."""
    import sparsecore_b200 as sl

    g = torch.Generator().manual_seed(3)
    rn = lambda *s: torch.randn(*s, generator=g).to(dtype).to(dev())  # noqa: E731
    y, r, w, b = rn(3, 50, 96), rn(3, 50, 96), 1 + 0.1 * rn(96), 0.1 * rn(96)
    head, t = 0.2 * rn(131, 96), torch.randint(0, 131, (3, 50), generator=g).to(dev())
    t[0, :7] = -100
    leaves = [v.clone().requires_grad_() for v in (y, r, w, b, head)]
    out, h = sl.residual_norm(*leaves[:4], scale=0.5)
    loss = sl.linear_cross_entropy(h, leaves[4], t)
    loss.backward()
    ref = [v.double().requires_grad_() for v in (y, r, w, b, head)]
    o64 = ref[1] + 0.5 * ref[0]
    o64 = o64 + (out.detach().double() - o64.detach())  # held in 16 bits
    h64 = torch.nn.functional.layer_norm(o64, (96,), ref[2], ref[3])
    h64 = h64 + (h.detach().double() - h64.detach())
    l64 = torch.nn.functional.cross_entropy((h64 @ ref[4].t()).view(-1, 131), t.view(-1))
    l64.backward()
    assert abs(float(loss.detach()) - float(l64.detach())) < 1e-5
    half = torch.finfo(dtype).eps / 2
    for got, want in zip(leaves, ref):
        assert got.grad.dtype == dtype
        assert float((got.grad.double() - want.grad).norm()) <= 3 * half * float(want.grad.norm())
    opt = sl.FusedAdamW(leaves, lr=1e-2, weight_decay=0.0)
    before = [v.detach().double() for v in leaves]
    opt.step()
    for v, v0, in zip(leaves, before):  # the first step moves every element by lr, against its gradient's sign
        moved = v0 - v.detach().double()
        gr = v.grad.double()
        want = 1e-2 * gr / (gr.abs() + 1e-8)
        assert bool(((moved - want).abs() <= 1e-2 * 1e-3 + half * (v0.abs() + 1e-2) * 2).all())
