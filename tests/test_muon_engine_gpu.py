"""The engines training with Muon: one step against 64-bit values, weight layouts refreshed, the
synchronisation modes, refusals."""
import os
import subprocess
import sys

import pytest
import torch

from distributed_machine_learning_amd.launch import launch
from support.muon_oracle import exact, rel

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
HERE = os.path.dirname(__file__)
WORKER = os.path.join(HERE, "_muon_worker.py")


def _backend(dtype="bf16", batch_norm=True, comm=None, **kw):
    from distributed_machine_learning_amd.config import TrainConfig
    from distributed_machine_learning_amd.engine.native_backend import NativeBackend
    torch.manual_seed(11)
    cfg = TrainConfig(batch_size=32, batch_norm=batch_norm, dtype=dtype, backend="native", lr=0.01,
                      optimizer="muon", muon_weight_decay=0.05, **kw)
    return NativeBackend(cfg, DEV, comm)


def _batch(nb, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.zeros(32, 32, 32, 4, dtype=nb.act_dtype, device=DEV)
    x[..., :3] = torch.randn(32, 32, 32, 3, generator=g).to(DEV)
    return x, torch.randint(0, 10, (32,), generator=g).to(DEV)


@pytest.mark.parametrize("precision", ["fp32", "fp16"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_engine_step_is_muon(dtype, precision):
    nb = _backend(dtype, muon_precision=precision)
    for step in range(2):
        p, m = nb.params.cpu().double(), nb.momentum.cpu().double()
        loss = nb.train_step(*_batch(nb, step))
        g = nb.grads[:p.numel()].cpu().double()
        assert bool(torch.isfinite(loss).all())
        named = {s.name: s for s in nb.slots}
        for at, rows, cols, f in nb._muon.matrices:
            s = slice(at, at + rows * cols)
            m[s] = 0.95 * m[s] + g[s]
            o = exact((g[s] + 0.95 * m[s]).view(rows, cols)).reshape(-1)
            want = (1 - 0.02 * 0.05) * p[s] - 0.02 * f * o
            # the update's share of the weights, off by 2^-8 at most with 11-bit factors and by 2^-15
            # with 22, and three roundings of the weights
            tol = 0.02 * f * float(o.norm()) * (2.0 ** -8 if precision == "fp16" else 2.0 ** -15)
            assert float((nb.params[s].cpu().double() - want).norm()) <= tol + 3 * 2.0 ** -24 * float(want.norm())
        for at, n in nb._muon.segments:
            s = slice(at, at + n)
            m[s] = 0.9 * m[s] + g[s] + 1e-4 * p[s]
            p[s] = p[s] - 0.01 * m[s]
            assert float((nb.params[s].cpu().double() - p[s]).norm()) <= 8 * 2.0 ** -24 * float(p[s].norm()) + 1e-12
        fc = named["fc1.weight"]
        assert (fc.offset, fc.numel) in nb._muon.segments
        assert rel(nb.momentum, m) <= 8 * 2.0 ** -24


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_engine_layouts_follow_the_update(dtype):
    """After a step the engine computes with the new weights: like a fresh one loaded with them."""
    nb = _backend(dtype, batch_norm=False)
    for step in range(2):
        nb.train_step(*_batch(nb, step))
    other = _backend(dtype, batch_norm=False)
    other.load_state_dict(nb.state_dict())
    x, t = _batch(nb, 9)
    a, b = nb.eval_batch(x, t), other.eval_batch(x, t)
    assert torch.equal(nb.logits(32), other.logits(32)) and torch.equal(a[0], b[0])
    # and the gradients (backward-data layouts) agree bit for bit too
    nb.momentum.zero_()
    for e in (nb, other):
        e.train_step(x, t)
    assert torch.equal(nb.grads, other.grads) and torch.equal(nb.params, other.params)


@pytest.mark.parametrize("sync", ["gather_scatter", "all_reduce", "ddp"])
def test_one_rank_of_any_mode_is_no_sync(sync):
    from distributed_machine_learning_amd.parallel.comm import RcclCommunicator
    port = 29640 + ["gather_scatter", "all_reduce", "ddp"].index(sync)
    comm = RcclCommunicator(f"127.0.0.1:{port}", 0, 1, 0, timeout_s=60)
    try:
        base = _backend()
        nb = _backend(sync=sync, comm=comm)
        for step in range(3):
            batch = _batch(base, step)
            assert float(base.train_step(*batch)) == float(nb.train_step(*batch))
        comm.guard_sync(30)
        assert torch.equal(nb.params, base.params) and torch.equal(nb.momentum, base.momentum)
        nb.close()
    finally:
        comm.destroy()


def test_priming_puts_the_state_back():
    nb = _backend()
    batch = _batch(nb)
    p, m = nb.params.clone(), nb.momentum.clone()
    nb.prime([batch], 3)
    assert torch.equal(nb.params, p) and torch.equal(nb.momentum, m)


def test_graph_mode_is_refused():
    with pytest.raises(ValueError, match="graph"):
        _backend(use_graph=True)


def test_engine_refuses_a_step_its_own_optimizer_would_fuse():
    nb = _backend()
    x, t = _batch(nb)
    nb.engine.set_fused_optimizer(True, 0.1, 0.9, 0.0, 1.0)
    with pytest.raises(RuntimeError, match="fused optimizer"):
        nb.engine.gradients_step(x.data_ptr(), t.data_ptr(), 32, nb._stream())


def _run(tmp_path, tag, nproc, extra, dtype):
    out = str(tmp_path / tag)
    args = ["--out", out, "--device", "cuda", "--backend", "native", "--dtype", dtype, "--transport",
            "loopback", "--batch-norm"] + extra
    rc = subprocess.call([sys.executable, WORKER] + args, timeout=300) if nproc == 1 else \
        launch(WORKER, args, nproc, timeout_s=300)
    assert rc == 0, tag
    return [torch.load(f"{out}.rank{r}", weights_only=True) for r in range(nproc)]


@pytest.mark.parametrize("dtype,wire", [("bf16", "fp32"), ("bf16", "bf16"), ("fp32", "fp32")])
def test_two_ranks_stay_bitwise_in_step(tmp_path, dtype, wire):
    ranks = _run(tmp_path, "two", 2, ["--sync", "ddp", "--batch-size", "8", "--iters", "3", "--bucket-cap-mb",
                                      "4", "--grad-comm-dtype", wire], dtype)
    for k in ranks[0]:
        if "running" not in k and "num_batches" not in k:
            assert torch.equal(ranks[0][k], ranks[1][k]), k
