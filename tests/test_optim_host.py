"""The optimizer's bookkeeping that needs no GPU: where a loaded state's counts
and learning rates end up, what copies keep, and what is refused before any
address is read."""
import copy
import pickle

import pytest
import torch


def _saved(capturable, counts=(5, 5, 2), torchs=False, lr=1e-3):
    """A state dict of three parameters as it comes from a file, on the host."""
    import sparsecore_b200 as sl

    params = [torch.zeros(4, requires_grad=True) for _ in counts]
    opt = torch.optim.AdamW(params, lr=lr) if torchs else sl.FusedAdamW(params, lr=lr, capturable=capturable)
    count = (lambda c: torch.tensor(c, dtype=torch.int64)) if capturable else int
    if torchs:
        count = lambda c: torch.tensor(float(c))  # noqa: E731
    for p, c in zip(params, counts):
        if c is None:
            continue
        opt.state[p].update(exp_avg=torch.ones(4), exp_avg_sq=torch.ones(4))
        if torchs or c != counts[0]:
            opt.state[p]["step"] = count(c)
    if not torchs:
        opt.param_groups[0]["step"] = count(counts[0])
    return opt.state_dict()


def test_counts_and_rates_go_to_the_parameters_device():
    import sparsecore_b200 as sl

    state = _saved(True, counts=(5, 5, 5), lr=torch.tensor(0.25))
    params = [torch.zeros(4, device="meta", requires_grad=True) for _ in range(3)]
    opt = sl.FusedAdamW(params, capturable=True)
    opt.load_state_dict(state)
    group = opt.param_groups[0]
    for v in (group["step"], group["lr"]):
        assert v.device.type == "meta" and v.numel() == 1
    assert group["step"].dtype == torch.int64


def test_a_counter_elsewhere_is_refused_before_it_is_used():
    from sparsecore_b200 import optim

    gpu0, host, z = torch.device("cuda", 0), torch.device("cpu"), torch.zeros
    for bad, dev in ((z((), dtype=torch.int64), gpu0), (z((), dtype=torch.int64, device="meta"), gpu0), (z(()), host),
                     (z(2, dtype=torch.int64), host), (3, gpu0)):
        with pytest.raises(ValueError, match="step"):
            optim._check_counter(bad, dev)
    optim._check_counter(z((), dtype=torch.int64), host)


def test_a_state_before_the_first_step_has_no_count():
    import sparsecore_b200 as sl

    make = lambda: sl.FusedAdamW([torch.zeros(4, requires_grad=True)])  # noqa: E731
    opt = make()
    opt.load_state_dict(make().state_dict())
    assert not opt.param_groups[0].get("step")


def test_counts_of_late_parameters_go_there_too():
    import sparsecore_b200 as sl

    params = [torch.zeros(4, device="meta", requires_grad=True) for _ in range(3)]
    opt = sl.FusedAdamW(params, capturable=True)
    opt.load_state_dict(_saved(True))
    own = opt.state[params[2]]["step"]
    assert own.device.type == "meta" and own.numel() == 1 and own.dtype == torch.int64
    assert "step" not in opt.state[params[0]] and "step" not in opt.state[params[1]]


@pytest.mark.parametrize("torchs", [False, True])
@pytest.mark.parametrize("was", [False, True])
@pytest.mark.parametrize("now", [False, True])
def test_counts_keep_their_values(was, now, torchs):
    import sparsecore_b200 as sl

    if torchs and was:
        pytest.skip("one form of torch's state is enough")
    for counts in ((5, 5, 2), (7, 7, 7), (3, None, 3), (4, 6, 6)):
        params = [torch.zeros(4, requires_grad=True) for _ in counts]
        opt = sl.FusedAdamW(params, capturable=now)
        opt.load_state_dict(_saved(was, counts, torchs))
        at = opt.param_groups[0]["step"]
        assert isinstance(at, torch.Tensor) == now
        for p, c in zip(params, counts):
            st = opt.state.get(p)
            if c is None:
                assert not st
                continue
            own = st.get("step", at)
            assert int(own) == c and isinstance(own, torch.Tensor) == now


@pytest.mark.parametrize("way", [copy.deepcopy, lambda o: pickle.loads(pickle.dumps(o))])
def test_copies_keep_what_a_step_needs(way):
    import sparsecore_b200 as sl

    p, q = torch.zeros(4, requires_grad=True), torch.zeros(4, requires_grad=True)
    opt = sl.FusedAdamW([p, q], lr=0.5, state_bits=8, capturable=True, seed=9, live={q: torch.zeros(4, dtype=torch.int32)})
    got = way(opt)
    assert (got.state_bits, got.capturable, got.seed) == (8, True, 9)
    new_p, new_q = got.param_groups[0]["params"]
    assert new_p is not p and list(got._columns()) == [new_q]
    with pytest.raises(ValueError):  # their own plans, not the first one's
        new_p.grad, new_q.grad = torch.ones(4), torch.ones(4)
        got.load_state_dict(_saved(False))
    assert got._plans == {} and got._plans is not opt._plans


def test_numbers_made_elsewhere_are_refused_before_they_are_read():
    from sparsecore_b200 import _native as N
    from sparsecore_b200 import optim

    n = int(N.load_library().sl_adamw_hyper_bytes())
    host, gpu0 = torch.device("cpu"), torch.device("cuda", 0)
    z = lambda k: torch.zeros(k, dtype=torch.uint8)  # noqa: E731
    optim._check_numbers(z(n), host)
    for bad, dev in ((z(n), gpu0), (z(n - 1), host), (z(2 * n)[::2], host), (z(n + 1)[1:], host)):
        with pytest.raises(ValueError, match="hyper"):
            optim._check_numbers(bad, dev)
    with pytest.raises(TypeError):
        optim._check_numbers(7, host)
