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


def test_a_workspace_inside_a_buffer_is_refused():
    """(Refused on the host, before any launch.)"""
    from distributed_machine_learning_amd.ops import native
    plan = native.MuonPlan([(0, 200, 300, 1.0)], [])
    count = 200 * 300
    behind = -(-4 * count // 256) * 256
    store = torch.zeros(plan.workspace_bytes + behind, dtype=torch.uint8, device=DEV)
    p, g, m = (torch.randn(count, device=DEV) for _ in range(3))
    inside = store[:4 * count].view(torch.float32)
    for args in ((inside, g, m), (p, inside, m), (p, g, inside)):
        with pytest.raises(ValueError, match="overlap"):
            native.muon_step_(plan, *args, 0.1, 0.9, 0.0, workspace=store)
    want = p.clone()
    native.muon_step_(plan, want, g.clone(), m.clone(), 0.1, 0.9, 0.0)
    inside.copy_(p)
    native.muon_step_(plan, inside, g, m, 0.1, 0.9, 0.0, workspace=store[behind:])
    assert torch.equal(inside, want)
