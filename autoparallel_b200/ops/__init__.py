"""Operator library (schemas + CPU reference + sm_100a kernels)."""
from .library import (  # noqa: F401
    attention,
    cross_entropy,
    dtype_cast,
    lib,
    ops,
    reference_impls,
    register_cuda_impl,
    rms_norm,
    rope,
    swiglu,
)
from . import moe_ops  # noqa: F401,E402  (registers the planner-visible MoE operators)
from .moe_ops import grouped_mm, moe_combine, moe_dispatch, moe_route, moe_slots  # noqa: F401,E402
from .mx4_ops import mx4_dequantize, mx4_linear, mx4_matmul, mx4_mm, mx4_mm_values, mx4_quantize, mx4_round  # noqa: F401,E402
