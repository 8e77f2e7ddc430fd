"""brickrec — MI355X-native scoring engine for the similar-sets / hybrid-recommendation hot
path of davidry777/Brickbrain-Rec-Engine.

Layers: ``_lib`` (ctypes over libbrickrec.so, the C-ABI in include/brickrec.h),
``engine.ItemIndex`` (device-resident index + batched search), and the drop-ins that keep
the reference's call signatures: ``recommenders`` (recommendation_system.py),
``constraints`` (hard_constraint_filter.py), ``semantic`` (NLPRecommender.semantic_search),
``api`` (FastAPI routes) and ``distributed`` (row-sharded index over RCCL).  ``fp8`` (8-bit rows and
their dense scores) and ``adjust`` (penalties, biases and masks on dense scores) work on torch CUDA
tensors; their names load when they are first used, so that the package needs no torch without them.
"""
from ._lib import BrickrecError  # noqa: F401
from .engine import ItemIndex, Predicate, bits_from_bool, bool_from_bits  # noqa: F401

_LAZY = {"Fp8Rows": "fp8", "quantize_rows": "fp8", "scores_fp8": "fp8", "adjust_scores": "adjust", "mask_words": "adjust"}


def __getattr__(name):
    if name in _LAZY:
        from importlib import import_module
        value = getattr(import_module("." + _LAZY[name], __name__), name)
        globals()[name] = value
        return value
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")


__version__ = "0.1.0"
