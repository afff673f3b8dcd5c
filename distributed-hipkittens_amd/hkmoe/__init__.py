"""hkmoe -- MI355X (gfx950) FP8 mixture-of-experts grouped-GEMM path.

Host-side Python layer over the ``tk_kernel`` pybind11 module, which in turn
wraps the C ABI of ``libhkmoe.so`` (include/hkmoe.h).  All compute runs in the
hand-written HIP kernels of that library; there is no CPU or PyTorch fallback:
importing this package raises ImportError when the native module is missing.

Entry points
  tk_kernel.dispatch_*      raw kernel entry points (reference calling style:
                            positional, caller-allocated torch tensors)
  hkmoe.MoELayer            owns e4m3 expert weights + scales, allocates the
                            workspace once per token count, runs the layer
  hkmoe.moe_forward_steps   the same layer one kernel at a time, returning
                            every intermediate (for parity tests)
  hkmoe.quant_*             device quantisers (per-tensor, 1x128, 128x128)
  hkmoe.rms_norm_quant      residual + norm + e4m3 operand in one pass
  hkmoe.router_logits       the router's product
  hkmoe.lora_add            adapters of many requests beside a projection
  hkmoe.MoEBlock            norm, router and layer; hkmoe.LoraLinear: projection
                            and adapters
  hkmoe.gemm_fp8 / gemm_mx  dense products, with bias, activation and residual
  hkmoe.layer_norm, route_topk, moe_permute, moe_combine
                            what stands around experts in training, with gradients
"""
import os
import sys

_PKG_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if _PKG_ROOT not in sys.path:
    sys.path.insert(0, _PKG_ROOT)

try:
    import tk_kernel  # noqa: E402
except ImportError as exc:  # pragma: no cover - exercised only on a broken tree
    raise ImportError(
        "hkmoe: native module tk_kernel is not built; run "
        "`python distributed-hipkittens_amd/hkmoe/build.py` (or __graft_entry__.build())"
    ) from exc

from .layer import (MoELayer, moe_forward, moe_forward_steps, pack_weights,  # noqa: E402
                    quant_block, quant_group, quant_tensor, gemm_fp8, quant_mx, mx_pack_scales, gemm_mx,
                    mx_pack_weight_scales, moe_forward_mx_steps, MoELayerMX)
from .block import LoraLinear, MoEBlock, lora_add, rms_norm_quant, router_logits  # noqa: E402
from .train import (MoEOrder, layer_norm, layer_norm_backward, layer_norm_forward, moe_combine,  # noqa: E402
                    moe_combine_backward, moe_combine_forward, moe_permute, moe_permute_backward,
                    moe_permute_forward, route_topk, route_topk_backward, route_topk_forward)

LIB_PATH = os.path.join(_PKG_ROOT, "libhkmoe.so")
SCALE_TENSOR = tk_kernel.SCALE_TENSOR
SCALE_BLOCK = tk_kernel.SCALE_BLOCK

__all__ = ["tk_kernel", "MoELayer", "moe_forward", "moe_forward_steps", "pack_weights", "quant_block",
           "quant_group", "quant_tensor", "gemm_fp8", "quant_mx", "mx_pack_scales", "gemm_mx",
           "mx_pack_weight_scales", "moe_forward_mx_steps", "MoELayerMX", "rms_norm_quant", "router_logits",
           "lora_add", "LoraLinear", "MoEBlock", "MoEOrder", "layer_norm", "layer_norm_forward",
           "layer_norm_backward", "route_topk", "route_topk_forward", "route_topk_backward", "moe_permute",
           "moe_permute_forward", "moe_permute_backward", "moe_combine", "moe_combine_forward",
           "moe_combine_backward", "LIB_PATH",
           "SCALE_TENSOR", "SCALE_BLOCK"]
