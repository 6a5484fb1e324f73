"""Optimizers: the bookkeeping base and the fused AdamW, momentum-SGD and Muon classes."""

from ._state import StateOptimizer
from .adamw import AdamWReferenceRN, AdamWReferenceSR
from .muon import MuonRN, MuonSR
from .sgd import SGDMReferenceRN, SGDMReferenceSR

__all__ = ["AdamWReferenceRN", "AdamWReferenceSR", "MuonRN", "MuonSR", "SGDMReferenceRN",
           "SGDMReferenceSR", "StateOptimizer"]
