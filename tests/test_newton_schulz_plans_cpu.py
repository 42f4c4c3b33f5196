"""Newton-Schulz plans without a GPU: the launches that are chosen stay within HIP's limits, one
that is refused raises, and the sizes of the GPU tests take every way through the kernels."""
import math
import random

import pytest
import torch

from distributed_machine_learning_amd.ops import native
from support.newton_schulz_cases import CASES, chosen

NS = native.ns_coefficients(5, native.NS_COEFFICIENTS)


def plan(batch, m, n, wide=True, coefficients=NS):
    return native._ns_plan(((m, n, batch, 0, n, m * n, 0, n, m * n, 0.0),), (), coefficients, 1e-7, wide)


@pytest.mark.parametrize("batch", [1, (1 << 21) - 1, 1 << 21, (1 << 21) + 1, 1 << 22, 5 * (1 << 21) + 3])
def test_large_batches_take_several_launches(batch):
    launches = plan(batch, 16, 16).launches
    assert {kernel for kernel, *_ in launches} == {"solo"}
    assert sum(blocks for _, _, blocks, *_ in launches) == batch
    assert all(0 < blocks * threads < 1 << 32 for _, _, blocks, threads, *_ in launches)


@pytest.mark.parametrize("batch,m,n", [(1, 1, 1 << 24), (1, 60000, 60000), (1, 1 << 14, 1 << 20), (4000, 200, 300),
                                       (20000, 1, 5000), (100, 2048, 2048)])
@pytest.mark.parametrize("wide", [True, False])
def test_launches_have_fewer_than_2_32_threads(batch, m, n, wide):
    for _, _, blocks, threads, _, joined in plan(batch, m, n, wide).launches:
        assert 0 < blocks * threads < 1 << 32 and joined * 8 * 256 < 1 << 32


def test_more_tiles_than_a_launch_takes_are_refused():
    for shape in [(1, 1 << 23, 1 << 23), (1, 1 << 24, 1 << 24), (1 << 22, 200, 5000)]:
        with pytest.raises(ValueError, match="too many"):
            plan(*shape)


@pytest.mark.skipif(torch.cuda.is_available(), reason="the launches would run")
@pytest.mark.parametrize("batch,m,n", [(2, 16, 16), (1, 200, 300), (1, 64, 3000)])
def test_a_refused_launch_raises(batch, m, n):
    """Without a device no launch is accepted."""
    p = plan(batch, m, n)
    ws = torch.empty(p.workspace_bytes + 256, dtype=torch.uint8)
    at = -(-ws.data_ptr() // 256) * 256
    x = torch.ones(batch, m, n)
    with pytest.raises(RuntimeError, match="newton_schulz"):
        p.orthogonalize(x.data_ptr(), torch.empty_like(x).data_ptr(), 0, at, p.workspace_bytes, 0)
    muon = native.MuonPlan([], [(0, 8)])
    with pytest.raises(RuntimeError, match="newton_schulz"):
        muon._plan.muon(*(x.data_ptr() // 16 * 16,) * 3, 0.1, 0.9, 0.0, True, 0.1, 0.9, 0.0, 1.0, 0, 0, 0)


@pytest.mark.parametrize("batch,m,n,wide,want", CASES, ids=lambda v: str(v) if not isinstance(v, dict) else "")
def test_the_way_of_every_case(batch, m, n, wide, want):
    """What the GPU tests of these sizes run (a changed estimate shows here)."""
    assert chosen(plan(batch, m, n, wide).launches) == want


def test_the_cases_take_every_way():
    """No plan of 6000 drawn sizes has a launch that no case has."""
    have = {(kernel, way, wide or kernel == "solo") for _, _, _, wide, want in CASES for kernel, way in want.items()}
    rng, one = random.Random(5), native.ns_coefficients(1, native.NS_COEFFICIENTS)

    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    met = set()
    for _ in range(6000):
        m = size(1, 6000)
        n, batch, wide = size(m, max(m, min(20000, 400_000_000 // m))), size(1, 32) if rng.random() < 0.5 else 1, rng.random() < 0.5
        if batch * m * n <= 3e7 and batch * m * m <= 3e7:
            p = native.lib().NewtonSchulzPlan([(m, n, batch, 0, n, m * n, 0, n, m * n, 0.0)], [], list(one), 1e-7, wide)
            met |= {(kernel, way, wide or kernel == "solo") for kernel, way in chosen(p.launches).items()}
    assert len(met) > 40 and met <= have, sorted(met - have)
