"""Muon updates at the edges of what the plan allows."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def test_a_plan_of_nothing_leaves_any_buffers_alone():
    from distributed_machine_learning_amd.ops import native
    for count in (0, 7):
        p, g, m = (torch.full((count,), float(i), device=DEV) for i in range(3))
        native.muon_step_(native.MuonPlan([], []), p, g, m, 0.1, 0.9, 0.1)
        assert all(torch.equal(t, torch.full_like(t, i)) for i, t in enumerate((p, g, m)))
