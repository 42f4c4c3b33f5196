"""Every way a Newton-Schulz plan chooses through the kernels, whole batches of it, against 64 bits."""
import pytest
import torch

from support.muon_oracle import exact, gradient, rel
from support.newton_schulz_cases import CASES
from support.newton_schulz_model import bound

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("dtype,tall", [(torch.float32, False), (torch.bfloat16, True), (torch.float16, False),
                                        (torch.float32, True)], ids=["fp32", "bf16-tall", "fp16", "fp32-tall"])
@pytest.mark.parametrize("batch,m,n,wide", [c[:4] for c in CASES])
def test_orthogonalize(batch, m, n, wide, dtype, tall):
    from distributed_machine_learning_amd.optim import orthogonalize
    x = gradient(m, n, m + n, (batch,)).to(dtype).to(DEV)
    if tall:
        x = x.transpose(1, 2).contiguous()
    y = orthogonalize(x, precision="fp32" if wide else "fp16")
    # one block per matrix has 22-bit factors whatever is asked for
    wide = wide or m * n == 1
    # all matrices of a few; of many the first, the last and those between whole and divided tiles
    for i in range(batch) if batch <= 8 else sorted({0, 1, batch // 2, batch - 3, batch - 2, batch - 1}):
        want = exact(x[i], device=DEV)
        off, most = rel(y[i], want), bound(x[i], want, dtype, wide, device=DEV)
        assert off <= most, i


@pytest.mark.parametrize("batch,m,n,wide", [c[:4] for c in CASES if c[0] > 1])
def test_matrices_of_a_batch_are_apart(batch, m, n, wide):
    """A matrix that is zero or not finite leaves the others' bits as they were, and calls repeat theirs."""
    from distributed_machine_learning_amd.optim import orthogonalize
    precision = "fp32" if wide else "fp16"
    x = gradient(m, n, m, (batch,)).to(DEV)
    good = orthogonalize(x, precision=precision)
    assert torch.equal(good, orthogonalize(x, precision=precision))
    x[batch // 2, m // 2, n // 3] = float("nan")
    x[0] = 0
    y = orthogonalize(x, precision=precision)
    assert torch.equal(y[0], x[0]) and bool(torch.isnan(y[batch // 2]).all())
    for i in range(1, batch):
        if i != batch // 2:
            assert torch.equal(y[i], good[i]), i


NS = (3.4445, -4.7750, 2.0315)


@pytest.mark.parametrize("steps,coefficients", [(1, NS), (2, NS), (3, NS), (4, NS), (6, NS), (8, NS), (4, (1.5, -0.5, 0.0)),
                                                (5, (1.875, -1.25, 0.375)), (2, (1.0, 0.0, 0.0)),
                                                (3, [(3.0, -3.2, 1.2), (1.875, -1.25, 0.375), (1.5, -0.5, 0.0)])])
@pytest.mark.parametrize("m,n", [(30, 50), (60, 3000), (200, 6000), (260, 300), (772, 3832)])
def test_steps_and_coefficients(m, n, steps, coefficients):
    from distributed_machine_learning_amd.optim import orthogonalize
    kw = dict(steps=steps, coefficients=coefficients)
    for dtype in (torch.float32, torch.bfloat16):
        x = gradient(m, n, 6).to(dtype).to(DEV)
        want = exact(x, device=DEV, **kw)
        off, most = rel(orthogonalize(x, **kw), want), bound(x, want, dtype, device=DEV, **kw)
        assert off <= most


@pytest.mark.parametrize("tall", [False, True])
@pytest.mark.parametrize("batch,m,n,wide", [c[:4] for c in CASES if c[0] <= 5])
def test_updates(batch, m, n, wide, tall):
    """The same ways where the last product writes weights: from zero by a step of one, the update is the
    direction itself.  (Each matrix has an entry of its own in the plan: a batch of one.)"""
    from distributed_machine_learning_amd.ops import native
    rows, cols = (n, m) if tall else (m, n)
    each = -(-rows * cols // 64) * 64
    matrices = [(i * each, rows, cols, 1.0) for i in range(batch)]
    p, g, buf = (torch.zeros(batch * each, device=DEV) for _ in range(3))
    inputs = gradient(rows, cols, m + n, (batch,)).to(DEV)
    for (at, *_), x in zip(matrices, inputs):
        g[at:at + rows * cols] = x.flatten()
    native.muon_step_(native.MuonPlan(matrices, [], precision="fp32" if wide else "fp16"), p, g, buf, 1.0, 0.0, 0.0)
    assert torch.equal(buf, g)
    for (at, *_), x in zip(matrices, inputs):
        want = exact(x, device=DEV)
        off, most = rel(-p[at:at + rows * cols].view(rows, cols), want), bound(x, want, wide=wide or m * n == 1, device=DEV)
        assert off <= most, at
