"""The package's checkpoints with FusedAdamW: a run goes on bit for bit, into a
model of the same or of another seed (other slots in every layer), with its
counts where the kernels read them."""
import numpy as np
import pytest
import torch

from gpu_helpers import dev
from test_gpu_checkpoint import _make, _masks, _step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", [0, 123])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
def test_resume_continues_bit_identically(tmp_path, seed, bits, capturable):
    import sparsecore_b200 as sl
    from sparsecore_b200 import checkpoint

    def make(s):
        model, algo, _ = _make(s)
        lr = torch.tensor(1e-2, device=dev()) if capturable else 1e-2
        return model, algo, sl.FusedAdamW(model, lr=lr, state_bits=bits, capturable=capturable)

    model, algo, opt = make(0)
    for i in range(5):
        _step(model, algo, opt, i)
    path = tmp_path / "ck.pt"
    checkpoint.save(path, model, opt, algo)
    ref = [_step(model, algo, opt, i) for i in range(5, 11)]
    model2, algo2, opt2 = make(seed)
    if seed == 0:
        _step(model2, algo2, opt2, 0)  # one that has moments and a table already
    checkpoint.load(path, model2, opt2, algo2)
    got = [_step(model2, algo2, opt2, i) for i in range(5, 11)]
    assert got == ref
    for (c1, v1, _), (c2, v2, _) in zip(_masks(model), _masks(model2)):
        assert np.array_equal(c1, c2) and np.array_equal(v1.view(np.int32), v2.view(np.int32))
    if capturable:
        group = opt2.param_groups[0]
        assert group["step"].device == group["lr"].device == dev() and int(group["step"]) == 11
