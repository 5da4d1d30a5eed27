"""Generic device helpers of the engine: top-k, RNG, reductions (mirrors the reference's
sklearn_numba_dpex/common package for the pieces the KMeans path uses), and beside them routing to
experts with what belongs to it, and products in 8-bit integers.

The expert and 8-bit calls come with an extension that is bound to one build of torch.  It is loaded when one of them is
first asked for, so that the helpers of the engine need nothing but the library."""
import importlib

from .random import create_xoroshiro128pp_states, get_random_raw  # noqa: F401
from .topk import topk, topk_idx  # noqa: F401

_LATER = dict.fromkeys(("combine_experts", "combine_experts_grad", "expert_slots", "route_topk", "route_topk_grad"), "experts")
_LATER.update(dict.fromkeys(("check_int8_waits", "int8_matmul", "quantize_rows"), "int8"))

__all__ = ["create_xoroshiro128pp_states", "get_random_raw", "topk", "topk_idx", *_LATER]


def __getattr__(name):
    if name in ("experts", "int8"):
        return importlib.import_module(f"{__name__}.{name}")
    if name not in _LATER:
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    value = globals()[name] = getattr(importlib.import_module(f"{__name__}.{_LATER[name]}"), name)
    return value


def __dir__():
    return sorted({*globals(), *__all__})
