"""CU masks for the control plane, and the head operators of the model zoo.

``linear``, ``layer_norm`` and ``distill_loss`` need torch and are imported
when first asked for: the plugin and the scheduler run without it.
"""
from importlib import import_module

from .cumask import CoreMaskAllocator, cus_for_percent, hsa_cu_mask_env  # noqa: F401

_OPERATORS = {"linear": "matmul", "layer_norm": "normalize", "distill_loss": "distill"}


def __getattr__(name):
    if name not in _OPERATORS:
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    value = getattr(import_module("." + _OPERATORS[name], __name__), name)
    globals()[name] = value
    return value
