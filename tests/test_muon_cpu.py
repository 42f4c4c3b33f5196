"""Muon and Newton-Schulz without a GPU: the torch form against 64-bit values, the plans' argument
checks, parameter selection, the command line and two gloo ranks."""
import math
import os
import subprocess
import sys

import pytest
import torch

from distributed_machine_learning_amd.launch import launch
from distributed_machine_learning_amd.ops import native
from distributed_machine_learning_amd.optim import Muon, orthogonalize
from distributed_machine_learning_amd.optim.muon import lr_factor, split_slots
from distributed_machine_learning_amd.parallel.flat import FlatModule
from support.muon_oracle import NS, exact, gradient, rel, tolerance

HERE = os.path.dirname(__file__)


class _Net(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.conv = torch.nn.Conv2d(3, 8, 3)
        self.body = torch.nn.Linear(8, 20)
        self.fc1 = torch.nn.Linear(20, 10)


@pytest.mark.parametrize("m,n", [(1, 1), (5, 3), (20, 33), (64, 64), (70, 200)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_orthogonalize_on_the_cpu(m, n, dtype):
    x = gradient(m, n, m + n).to(dtype)
    y = orthogonalize(x)
    assert y.shape == x.shape and y.dtype == dtype
    assert rel(y, exact(x)) <= tolerance(x, True, dtype)
    batch = torch.stack([x, torch.zeros_like(x), 2 * x])
    yb = orthogonalize(batch)
    # (a batched product may sum in another order: held to the same bound, not to the same bits)
    assert rel(yb[0], exact(x)) <= tolerance(x, True, dtype) and bool((yb[1] == 0).all())


def test_the_iteration_sends_singular_values_near_one():
    x = torch.randn(40, 90, generator=torch.Generator().manual_seed(0))
    s = torch.linalg.svdvals(exact(x))
    assert 0.6 < float(s.min()) and float(s.max()) < 1.25


def test_steps_of_the_definition_match_the_polynomial_of_the_singular_values():
    """The oracle itself, against another way to compute the map."""
    x = gradient(12, 30, 4).double()
    u, s, v = torch.linalg.svd(x / (x.norm() + 1e-7), full_matrices=False)
    for a, b, c in [NS] * 5:
        s = a * s + b * s ** 3 + c * s ** 5
    assert rel(exact(x), u @ torch.diag(s) @ v) <= 1e-12


def test_orthogonalize_refusals():
    x = torch.randn(4, 5)
    with pytest.raises(TypeError):
        orthogonalize(x.double())
    with pytest.raises(ValueError):
        orthogonalize(x[0])
    with pytest.raises(ValueError):
        orthogonalize(x, steps=0)
    with pytest.raises(ValueError):
        orthogonalize(x, steps=65)
    with pytest.raises(ValueError):
        orthogonalize(x, steps=2, coefficients=[(1.0, 2.0, 3.0)])
    with pytest.raises(ValueError):
        orthogonalize(x, precision="fp8")
    with pytest.raises(ValueError, match="GPU"):
        native.newton_schulz(x)


def test_orthogonalize_takes_leaves_and_detaches():
    x = torch.randn(4, 5, requires_grad=True)
    assert not orthogonalize(x).requires_grad


def _plan(matrices=((0, 4, 6, 1.0),), segments=(), **kw):
    return native.MuonPlan(matrices, segments, **kw)


def test_plan_refusals():
    for bad in [((0, 4, 6, 1.0), (20, 4, 6, 1.0)), ((-1, 4, 6, 1.0),), ((0, 0, 6, 1.0),)]:
        with pytest.raises(ValueError):
            _plan(bad)
    with pytest.raises(ValueError):
        _plan(segments=((10, 4),))
    with pytest.raises(ValueError):
        _plan(precision="bf16")
    with pytest.raises(ValueError, match="grow past 8"):
        _plan(coefficients=(3.0, 3.0, 3.0))
    with pytest.raises(ValueError):
        _plan(coefficients=(float("nan"), 0.0, 0.0))
    with pytest.raises(ValueError):
        _plan(eps=-1.0)
    with pytest.raises(ValueError):
        _plan(eps=float("nan"))
    with pytest.raises(ValueError):
        _plan(((0, 1, (1 << 24) + 1, 1.0),))
    with pytest.raises(ValueError):
        _plan(steps=0)


def test_plan_of_nothing_and_of_vectors():
    assert _plan((), ()).elems == 0
    p = _plan((), ((8, 4), (64, 0)))
    assert p.elems == 12 and p.segments == ((8, 4),)


def test_plan_extent_and_workspace():
    p = _plan(((64, 512, 4608, 1.0), (0, 4, 6, 1.0)), ((30, 10),))
    assert p.elems == 64 + 512 * 4608
    # two copies of Y in two 2-byte planes at least, and no more than a few times that
    assert 8 * 512 * 4608 <= p.workspace_bytes <= 40 * 512 * 4608


def test_lr_factor():
    assert lr_factor(512, 4608) == 1.0 and lr_factor(400, 100) == 2.0
    assert math.isclose(lr_factor(400, 100, "match_rms_adamw"), 4.0)
    with pytest.raises(ValueError):
        lr_factor(1, 1, "adam")


def test_split_slots():
    flat = FlatModule(_Net())
    matrices, segments = split_slots(flat.slots, None, "original")
    at = {s.name: s for s in flat.slots}
    assert [(o, r, c) for o, r, c, _ in matrices] == [(at["conv.weight"].offset, 8, 27),
                                                      (at["body.weight"].offset, 20, 8)]
    assert (at["fc1.weight"].offset, 200) in segments and len(segments) == 4
    matrices, _ = split_slots(flat.slots, ["body.weight"], "original")
    assert [(r, c) for _, r, c, _ in matrices] == [(8, 27), (10, 20)]
    with pytest.raises(ValueError, match="nowhere"):
        split_slots(flat.slots, ["nowhere"], "original")
    with pytest.raises(ValueError):
        Muon(_Net(), precision="half")
    with pytest.raises(ValueError):
        Muon(_Net(), adjust_lr_fn="none")


@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step_on_the_cpu(nesterov):
    torch.manual_seed(1)
    opt = Muon(_Net(), lr=0.05, momentum=0.9, weight_decay=0.1, nesterov=nesterov)
    p, m = opt.flat.params.double(), opt.buf.double()
    for step in range(3):
        opt.zero_grad()
        for s in opt.flat.slots:
            opt.flat.grads[s.offset:s.end] = torch.randn(s.numel)
        g = opt.flat.grads.double() * 0.25
        opt.step(grad_scale=0.25)
        for at, rows, cols, f in opt.matrices:
            s = slice(at, at + rows * cols)
            m[s] = 0.9 * m[s] + g[s]
            o = exact((g[s] + 0.9 * m[s] if nesterov else m[s]).view(rows, cols))
            p[s] = (1 - 0.05 * 0.1) * p[s] - 0.05 * f * o.reshape(-1)
        for at, n in opt.segments:
            s = slice(at, at + n)
            m[s] = 0.9 * m[s] + g[s] + 1e-4 * p[s]
            p[s] = p[s] - 0.1 * m[s]
        assert rel(opt.flat.params, p) <= 1e-5 and rel(opt.buf, m) <= 1e-6
    assert opt.steps == 3


def test_command_line_trains_with_muon():
    cmd = [sys.executable, os.path.join(HERE, "..", "part1", "main.py"), "--device", "cpu", "--iters", "2",
           "--batch-size", "2", "--train-size", "8", "--test-size", "4", "--no-summary", "--no-eval",
           "--optimizer", "muon", "--muon-lr", "0.01"]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr
    assert "Optimizer: muon, lr=0.01, momentum=0.95, weight_decay=0.0, precision=fp32" in r.stdout


def test_two_ranks_stay_in_step(tmp_path):
    out = str(tmp_path / "muon")
    rc = launch(os.path.join(HERE, "_muon_worker.py"),
                ["--out", out, "--sync", "ddp", "--iters", "2", "--batch-size", "2"], 2, timeout_s=300)
    assert rc == 0
    a, b = (torch.load(f"{out}.rank{r}", weights_only=True) for r in range(2))
    assert all(torch.equal(a[k], b[k]) for k in a)
