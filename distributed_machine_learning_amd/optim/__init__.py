from .fused_sgd import FusedSGD  # noqa: F401
from .muon import Muon, orthogonalize  # noqa: F401
