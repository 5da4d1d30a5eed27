"""The C++ side of the expert and 8-bit calls (csrc/torch_calls.cpp): checks, allocation and launch on torch
tensors.  Like the library itself it has no fallback."""
from .. import _cabi  # noqa: F401  (loads the library that the extension calls)

try:
    from .._torch_calls import (combine_experts, combine_experts_grad, expert_slots, int8_matmul,  # noqa: F401
                                quantize_rows, route_topk, route_topk_grad)
except ImportError as exc:
    raise ImportError(f"{exc}: the calls on torch tensors are not built. Run "
                      "`python -m sklearn_numba_dpex_b200.build` in a checkout, or install with "
                      "`pip install --no-build-isolation .`; there is no fallback.") from exc
