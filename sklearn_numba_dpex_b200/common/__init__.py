"""Generic device helpers of the engine: top-k, RNG, reductions (mirrors the reference's
sklearn_numba_dpex/common package for the pieces the KMeans path uses), and beside them routing to
experts with what belongs to it, and products in 8-bit integers."""
from .experts import (combine_experts, combine_experts_grad, expert_slots, route_topk,  # noqa: F401
                      route_topk_grad)
from .int8 import check_int8_waits, int8_matmul, quantize_rows  # noqa: F401
from .random import create_xoroshiro128pp_states, get_random_raw  # noqa: F401
from .topk import topk, topk_idx  # noqa: F401
