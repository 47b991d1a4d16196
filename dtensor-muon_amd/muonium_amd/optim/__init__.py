from .adamw import AdamW, AdamWFp8
from .algorithms import (
    BufferSpec,
    MuonAlgorithm,
    get_algorithm,
    register_muon_algorithm,
    registered_algorithms,
)
from .lp_state import OptimStateFp8
from .optim import Muon
from .optim_lp import Muon4bit, Muon8bit, MuonFp8, MuonLP

__all__ = [
    "AdamW",
    "AdamWFp8",
    "BufferSpec",
    "Muon",
    "Muon4bit",
    "Muon8bit",
    "MuonAlgorithm",
    "MuonFp8",
    "MuonLP",
    "OptimStateFp8",
    "get_algorithm",
    "register_muon_algorithm",
    "registered_algorithms",
]
