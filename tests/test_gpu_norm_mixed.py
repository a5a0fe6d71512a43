"""residual_norm where a 16-bit block output meets a 32-bit stream, over the
widths at which its rows are spread and held differently.  Tolerances as in
test_gpu_norm."""
import pytest
import torch

from gpu_helpers import dev
from test_gpu_norm import _case, _check

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("D", [2048, 2056, 2500, 4000, 4096, 4104])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("post", [False, True])
def test_a_gate_a_row_over_a_32_bit_stream(D, dtype, post):
    for kind in ("layer", "rms"):
        _check(_case(37, D, dtype, D, kind=kind, rdtype=torch.float32, gate=(37,), post=post))


@gpu
@pytest.mark.parametrize("D", [2056, 4096])
def test_one_row_and_sequences_of_one_row(D):
    """A gate that belongs to one row only is a gate a row, however it is given."""
    import sparsecore_b200 as sl

    _check(_case(1, D, torch.bfloat16, D, rdtype=torch.float32, gate=(1,), post=True))
    c = _case(5, D, torch.bfloat16, D + 1, rdtype=torch.float32, gate=(5,), post=True)
    names = ("y", "r", "w", "b", "gate", "pw", "pb")

    def grads(shape, gshape):
        leaf = {k: c[k].clone().requires_grad_() for k in names}
        out, h = sl.residual_norm(leaf["y"].view(shape), leaf["r"].view(shape), leaf["w"], leaf["b"], gate=leaf["gate"].view(gshape),
                                  post_weight=leaf["pw"], post_bias=leaf["pb"])
        return torch.autograd.grad((out, h), [leaf[k] for k in names], (c["dout"].view(shape), c["dh"].view(shape)))

    for a, b in zip(grads((5, D), (5, D)), grads((5, 1, D), (5, 1, D))):
        assert torch.equal(a.reshape(-1), b.reshape(-1))


@gpu
@pytest.mark.parametrize("wdtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("gate", [None, (1,), (3,), (33,)])
def test_vectors_of_either_type_over_a_32_bit_stream(wdtype, gate):
    for D in (1000, 3000):
        _check(_case(33, D, torch.float16, D, rdtype=torch.float32, wdtype=wdtype, gate=gate, post=True))
    _check(_case(33, 4096, torch.float16, 7, rdtype=torch.float32, wdtype=wdtype, gate=gate))
