"""The CPU sample keeps to its time: a host on which the full batch would take
minutes a step takes fewer sequences and says so, and an arm without the
reference's kernels says that instead of timing something else."""
import importlib.util
import json
import os
import subprocess
import sys
import time

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def bench():
    spec = importlib.util.spec_from_file_location("bench_under_test", os.path.join(REPO, "bench.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


class _Kernels:
    kind = "port"


@pytest.fixture
def slow_host(bench, monkeypatch):
    """A host on which a step takes `pace` seconds a sequence, on a clock of its own."""
    import torch

    from oracle import ref_arm

    clock = {"now": 0.0, "pace": 25.0}

    class Workload:
        unit, data, units_of = "tokens/s", "synthetic", 512

        def __init__(self, name, device, rank, linear=None, batch=None):
            n = batch or 32
            self.batch, self.units, self.config = (torch.zeros(n, 3),), n * self.units_of, {"global_batch": 32}
            self.model = None
            self.opt = type("Opt", (), {"zero_grad": lambda s: None, "step": lambda s: None})()

        def loss_fn(self, model, batch):
            clock["now"] += clock["pace"] * batch[0].shape[0]
            return torch.ones((), requires_grad=True) * 1.0

    monkeypatch.setattr(bench, "Workload", Workload)
    monkeypatch.setattr(ref_arm, "kernels", lambda: _Kernels)
    monkeypatch.setattr(ref_arm, "linear_factory", lambda kern: None)
    monkeypatch.setattr(time, "perf_counter", lambda: clock["now"])
    return clock


def test_a_slow_host_takes_fewer_sequences(bench, slow_host):
    got = bench.cpu_sample("cfg5", None, 1, 2, budget_s=100.0, min_steps=2)
    assert got["_config"]["global_batch"] == 1 and got["steps"] == 2 and "1 of its 32" in got["sample"]
    assert got["value"] == pytest.approx(512 / 25.0, rel=1e-3)
    assert slow_host["now"] <= 25.0 + 100.0


def test_a_quick_host_takes_the_full_batch(bench, slow_host):
    slow_host["pace"] = 0.3
    got = bench.cpu_sample("cfg5", None, 1, 20, budget_s=200.0, min_steps=3)
    assert got["_config"]["global_batch"] == 32 and got["steps"] == 20 and "of the full cfg5 batch" in got["sample"]
    slow_host["pace"] = 1.0  # 32 s a step: fewer steps, not fewer sequences
    got = bench.cpu_sample("cfg5", None, 1, 20, budget_s=200.0, min_steps=3)
    assert got["_config"]["global_batch"] == 32 and got["steps"] == 6


def test_the_reference_arm_times_nothing_else():
    from oracle import ref_arm

    if ref_arm.kernels().kind == "reference":
        pytest.skip("the reference's kernels are built here")
    res = subprocess.run([sys.executable, os.path.join(REPO, "bench.py"), "--impl", "reference", "--steps", "20"], cwd=REPO,
                         capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr[-2000:]
    line = json.loads(res.stdout.strip().splitlines()[-1])
    assert line["impl"] == "reference" and line["unavailable"] and "value" not in line
