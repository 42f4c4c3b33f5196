"""The optimizer of a training run is the one that its configuration names."""
import pytest
import torch

from distributed_machine_learning_amd.config import TrainConfig
from distributed_machine_learning_amd.engine.native_backend import NativeBackend
from distributed_machine_learning_amd.engine.torch_backend import TorchBackend
from distributed_machine_learning_amd.optim import Muon


@pytest.mark.parametrize("backend", [NativeBackend, TorchBackend])
@pytest.mark.parametrize("name", ["Muon", "adam", ""])
def test_unknown_optimizers_are_refused(backend, name):
    """(They trained with SGD.  The native backend refuses before it touches a device.)"""
    with pytest.raises(ValueError, match="optimizer"):
        backend(TrainConfig(optimizer=name, dtype="fp32"), torch.device("cuda" if backend is NativeBackend else "cpu"), None)


def test_known_ones_are_taken():
    for name, kind in (("sgd", torch.optim.SGD), ("muon", Muon)):
        assert isinstance(TorchBackend(TrainConfig(optimizer=name, dtype="fp32"), torch.device("cpu"), None).optimizer, kind)
