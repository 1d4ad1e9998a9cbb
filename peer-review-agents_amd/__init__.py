"""MI355X-native (gfx950) Expert-Threshold MoE token-dispatch path.

Import with ``importlib.import_module("peer-review-agents_amd")`` (the
directory name is not a Python identifier).  Kernels live in csrc/ and are
built into libetmoe.so by build.py; the host API is in expert_threshold.py (the
dispatch path), norm.py (layer norm), optimizer.py (AdamW, the gradient norm)
and w4.py (products with 4-bit weights), and ops.py registers
the path as PyTorch operators (torch.ops.etmoe.*).
"""
from ._lib import BLOCK_HEADER_PATH, ETMoEError, LIB_PATH, header_symbols, lib  # noqa: F401
from . import ops  # noqa: F401  (registers torch.ops.etmoe.*)
from .expert_threshold import (  # noqa: F401
    ExpertThresholdRouter,
    RoutingPlan,
    combine,
    combine_autograd,
    combine_backward,
    combine_backward_workspace_bytes,
    dispatch,
    dispatch_autograd,
    dispatch_backward,
    expert_gemm,
    expert_gemm_fp8,
    expert_gemm_input_grad,
    expert_gemm_weight_grad,
    expert_weight_transpose,
    route,
    route_update,
    route_workspace_bytes,
    router_logits,
    router_route,
    router_route_workspace_bytes,
    router_weight_grad,
    swiglu,
    swiglu_backward,
    threshold_update_,
    threshold_workspace_bytes,
)
from .norm import (  # noqa: F401
    layer_norm,
    layer_norm_autograd,
    layer_norm_backward,
    layer_norm_backward_workspace_bytes,
)
from .optimizer import (  # noqa: F401
    ADAMW8_BLOCK,
    AdamW,
    adamw8_scales,
    adamw8_step_,
    adamw_step_,
    grad_norm,
)
from .w4 import (  # noqa: F401
    W4Weight,
    expert_gemm_w4,
    linear_w4,
    pack_w4,
    quantize_w4,
    unpack_w4,
)
